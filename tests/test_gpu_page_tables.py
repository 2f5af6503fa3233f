"""Page tables, slots and positions of a step, against the same rules a request and a token at a time."""
import numpy as np
import pytest

import morello_amd as M

pytestmark = pytest.mark.gpu


def by_hand(op, cached, added, free, count, table):
    requests, width, page, pages, tokens, capacity = (getattr(op._c, n) for n in ("requests", "table_width", "page_size", "pages", "tokens", "free_pages"))
    count = min(max(count, 0), capacity)
    table = table.copy()
    starts, lengths, slots, positions, drawn = [0], [], np.full(tokens, -1), np.zeros(tokens, int), 0
    for r in range(requests):
        c, n = max(int(cached[r]), 0), max(int(added[r]), 0)
        n = min(n, tokens - starts[-1])
        have, need = min(-(-c // page), width), min(-(-(c + n) // page), width)
        for column in range(have, need):
            table[r, column] = free[count - 1 - drawn] if drawn < count else -1
            drawn += 1
        for i in range(n):
            p = c + i
            positions[starts[-1] + i] = min(p, 2 ** 31 - 1)
            if p // page < width and 0 <= table[r, p // page] < pages:
                slots[starts[-1] + i] = table[r, p // page] * page + p % page
        starts.append(starts[-1] + n)
        lengths.append(min(c + n, 2 ** 31 - 1))
    return [x.astype(np.int32) for x in (table, np.array(starts), np.array(lengths), slots, positions, np.array([count - min(drawn, count), drawn - min(drawn, count)]))]


def run(op, cached, added, free, count, table, times=1):
    c = op._c
    host = [np.asarray(x, np.int32) for x in (cached, added, free if len(free) else [0], [count])] + [table.astype(np.int32)] + [
        np.full(n, -77, np.int32) for n in (c.requests + 1, c.requests, c.tokens, c.tokens, 2)]
    bufs = [M.DeviceBuffer.from_numpy(x) for x in host]
    for _ in range(times):
        op.run_device([b.ptr for b in bufs])
    got = [bufs[i].to_numpy(np.int32, host[i].shape) for i in range(4, 10)]
    for b in bufs:
        b.free()
    return got


def check(page, lengths, tokens=None, width=None, pages=None, count=None, spare=5, times=1, seed=0, bad=False):
    rng = np.random.default_rng(seed)
    cached, added = np.array([c for c, _ in lengths]), np.array([n for _, n in lengths])
    have = -(-np.maximum(cached, 0) // page)
    wanted = int((-(-(np.maximum(cached, 0) + np.maximum(added, 0)) // page) - have).sum())
    pages = pages or int(have.clip(max=width).sum()) + wanted + spare
    width = width or int((-(-(np.maximum(cached, 0) + np.maximum(added, 0)) // page)).max()) + 2
    ids = rng.permutation(pages)
    table = np.full((len(lengths), width), -1, np.int64)
    at = 0
    for r, h in enumerate(have.clip(max=width)):
        table[r, :h] = ids[at:at + h]
        at += h
    table[:, -1] = np.where(table[:, -1] < 0, -9, table[:, -1])
    free = ids[at:]
    if bad:   # numbers outside the cache on the list and in the table: their tokens have no slot
        free = np.where(np.arange(len(free)) % 3 == 0, pages + 5, free)
        table[::2] = np.where(table[::2] >= 0, pages, table[::2])
    count = len(free) if count is None else count
    op = M.PageTables(len(lengths), width, page, pages, tokens or max(1, int(np.maximum(added, 0).sum()) + 4), len(free))
    want = by_hand(op, cached, added, free, count, table)
    for name, g, w in zip(("table", "starts", "lengths", "slots", "positions", "free left"), run(op, cached, added, free, count, table, times), want):
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5].tolist())


@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_mixed_lengths(gpu, page):
    rng = np.random.default_rng(page)
    check(page, [(int(c), int(n)) for c, n in zip(rng.integers(0, 200, 37), rng.choice([0, 1, 1, 1, 2, 15, 16, 17, 130], 37))])


def test_one_token_and_none(gpu):
    check(16, [(0, 1)])
    check(16, [(16, 1)])
    check(16, [(15, 1)])
    check(16, [(0, 0)])
    check(16, [(33, 0), (0, 0), (5, 0)])
    check(16, [(0, 0), (0, 3), (0, 0), (0, 0), (16, 17), (0, 0)])


def test_many_requests_and_tokens(gpu):
    """Requests past a pass of 1024, tokens past a workgroup's 1024, runs of requests without tokens on either side of both."""
    rng = np.random.default_rng(3)
    lengths = [(int(c), int(n)) for c, n in zip(rng.integers(0, 60, 2500), rng.choice([0, 0, 0, 1, 1, 3], 2500))]
    lengths[1020:1030] = [(5, 0)] * 10
    check(16, lengths)
    check(16, [(0, 5000), (3, 1), (100, 1023), (1, 1), (7, 0), (0, 1024)])
    check(8, [(0, 1024), (0, 1024), (0, 1)])


def test_run_again_gives_the_same(gpu):
    check(16, [(40, 1), (0, 100), (31, 2)], times=3)


def test_a_list_that_runs_out(gpu):
    for count in (0, 1, 5, -3, 1000):
        check(16, [(10, 30), (16, 16), (0, 100), (7, 1)], count=count)


def test_rows_and_columns_that_run_out(gpu):
    check(16, [(10, 30), (16, 16), (0, 100), (7, 1)], tokens=50)
    check(16, [(10, 30), (16, 16), (0, 100), (7, 1)], tokens=30)
    check(16, [(10, 30), (100, 16), (0, 100), (47, 2), (48, 1)], width=3)


def test_negative_lengths_and_pages_outside(gpu):
    check(16, [(-5, 3), (20, -7), (-1, -1), (0, 20)])
    check(16, [(40, 20), (40, 20), (3, 40), (15, 2)], bad=True)


def test_lengths_whose_sum_passes_32_bits(gpu):
    check(16, [(2 ** 31 - 1, 40), (10, 40), (2 ** 31 - 20, 30)], width=4, pages=32, tokens=110)
    op = M.PageTables(3, 4, 16, 32, 100, 4)
    free, table = np.arange(4), np.full((3, 4), -1)
    added = [2 ** 31 - 1] * 3
    for g, w in zip(run(op, [0, 0, 0], added, free, 4, table), by_hand(op, [0, 0, 0], added, free, 4, table)):
        assert np.array_equal(g, w)


def test_refused_pointers(gpu):
    """A written parameter over another: workgroups would read what others have written."""
    op = M.PageTables(3, 4, 16, 32, 100, 5)
    sizes = [3, 3, 5, 1, 12, 4, 3, 100, 100, 2]
    buf = M.DeviceBuffer(4 * 4096)
    at = [buf.ptr + 1024 * i for i in range(10)]
    for i in range(10):
        with pytest.raises(M.MorelloError) as err:
            op.run_device([None if j == i else p for j, p in enumerate(at)])
        assert err.value.status == 6
        for j in range(max(4, i + 1), 10):
            for over in (at[j], at[j] + 4 * (sizes[j] - 1), at[j] - 4 * (sizes[i] - 1)):   # on it, its last entry, its first
                with pytest.raises(M.MorelloError) as err:
                    op.run_device([over if k == i else p for k, p in enumerate(at)])
                assert err.value.status == 3 and "overlaps" in str(err.value)
    buf.free()
    check(16, [(3, 2), (0, 1)])   # (buffers side by side are fine)
