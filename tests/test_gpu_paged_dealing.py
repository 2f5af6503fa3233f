"""Attention over pages where workgroups' shares are long: tiles cut in the middle, pieces of more blocks than page numbers are fetched at a time, scores that outgrow
their reference late in a piece, requests of more tokens than the table holds keys.  Each case first makes sure, on the host, that its sizes come to that."""
import copy
import re

import numpy as np
import pytest

import morello_amd as M
from paged_util import DTYPE, POISON, STORED, Batch, as_f64, values

pytestmark = pytest.mark.gpu


def form_of(op):
    """(rows of a tile, keys of a block, workgroups, least, second, overhead) of a call that shares work out, by its plan and the kernels' numbers."""
    step = op.plan().steps[0]
    assert op.plan().kernels[-1].startswith("k_paged_attn_merge")
    qb, dims = re.search(r"QB = (\d)", step.kernel), int(re.search(r"D = (\d+)", step.kernel).group(1))
    if qb:
        return 16 * int(qb.group(1)), 32, step.grid[0], 4, 12, 3
    return 128, 64, step.grid[0], 8, 7, 7 if dims <= 64 else 4


def deal(batch, op, window=0):
    """-> (the few tiles' way?, of each workgroup its pieces (request, head, tile, first block, one behind the last, blocks of the tile), tiles whose lengths have stopped to grow):
    what morello_amd/csrc/paged_line.h and the kernels' Worker do."""
    bq, block, workers, least, second, overhead = form_of(op)
    group, capacity = batch.q_heads // batch.kv_heads, batch.width * batch.page
    step, more, slope = bq // group + 1, 4 + overhead, bq * 256 // group // block + 1
    tiles = []   # request, blocks, length on the line, of one head
    stopped = 0
    line = total = few_blocks = 0
    for r in range(batch.requests):
        n, length = int(batch.starts[r + 1] - batch.starts[r]), int(batch.totals[r])
        count = -(-n * group // bq)
        first, most = (min(max(length - n, 0), capacity) + step) // block + more, (min(window or capacity, capacity) + step) // block + more
        grown = (most - first) * 256 // slope + 1 if first < most else 0
        before = lambda t: min(t, grown) * first + (min(t, grown) * max(min(t, grown) - 1, 0) // 2 * slope >> 8) + max(t - grown, 0) * most
        mine = []
        for t in range(count):
            last, at = length - n + (min(n * group, (t + 1) * bq) - 1) // group, length - n + t * bq // group
            end = min(max(last + 1, 0), capacity, max(length, 0))
            begin = min(max(at - window + 1, 0), end) if window else 0
            mine.append((r, (end - 1) // block - begin // block + 1 if end > begin else 0, before(t + 1) - before(t)))
        stopped += max(count - grown, 0) if grown else 0
        tiles.append(mine)
        line, total = line + before(count) * batch.kv_heads, total + count * batch.kv_heads
        few_blocks += count * max([b for _, b, _ in mine] + [1]) * batch.kv_heads
    share, few = max(line // workers + (line % workers != 0), 1), False
    if total < workers:   # (a window's most blocks are rounded up a little more there; no case here is so near)
        single = -(--(-few_blocks // (workers - total)) // least) * least
        few = single <= share + second
        share = single if few else share
    pieces, at = [[] for _ in range(workers)], 0
    for mine in tiles:
        for head in range(batch.kv_heads):
            for tile, (r, blocks, length) in enumerate(mine):
                if few:
                    length = -(-max(b for _, b, _ in mine) // share) * share
                for w in range(at // share, (at + length - 1) // share + 1):
                    b0, b1 = min(max(w * share - at, 0), blocks), min((w + 1) * share - at, blocks)
                    if b0 < b1:
                        pieces[w].append((r, head, tile, b0, b1, blocks))
                at += length
    return few, pieces, stopped


def sample(batch, tokens):
    """Tokens of a batch as requests of their own, each with the keys up to its place: their rows are the batch's."""
    of = np.searchsorted(batch.starts, tokens, side="right") - 1
    b = copy.copy(batch)
    b.requests = b.tokens = len(tokens)
    b.starts = np.arange(len(tokens) + 1, dtype=np.int32)
    b.totals = (batch.totals[of] - (batch.starts[of + 1] - tokens) + 1).astype(np.int32)
    b.table, b.q64 = batch.table[of], batch.q64[tokens]
    return b


def check_tokens(batch, got, tokens, window=0, scale=None):
    """Those tokens' rows against the formula, all others for being numbers, or untouched behind the last."""
    g, end = as_f64(batch.dtype, got), int(batch.starts[-1])
    assert np.isfinite(g[:end]).all() and (g[end:] == 5).all()
    sample(batch, np.asarray(tokens)).check(got[tokens], window, scale)


def check_counts(batch, op, window=0):
    """Queries of zero, so that every key seen weighs 1, and values that are 1 in the dim that their page's number names and 0 elsewhere: each row is the share of its keys on
    the pages of each dim, all of them whole numbers below 2^24 until the quotient.  That is the reciprocal of 32 bits, a product and a rounding to the result's type.  A block of
    keys that is left out or taken twice is 1 to 3 % of a dim or more."""
    b = copy.copy(batch)
    one = {"bf16": np.uint16(0x3f80), "f32": np.float32(1)}[b.dtype]
    b.q = np.where(np.arange(b.tokens)[:, None, None] < b.starts[-1], STORED[b.dtype](0), b.q).astype(b.q.dtype)
    cache = b.values.transpose(0, 2, 1, 3) if b.heads_first else b.values
    poisoned = ~np.isfinite(as_f64(b.dtype, cache[:, :, 0, 0]))
    cache = np.zeros_like(cache)
    for page in range(b.pages):
        cache[page, :, :, page % b.dim] = one
    cache[poisoned] = POISON[b.dtype]
    b.values = np.ascontiguousarray(cache.transpose(0, 2, 1, 3)) if b.heads_first else cache
    got = as_f64(b.dtype, b.run(op))
    half = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}[b.dtype]
    for r in range(b.requests):
        start, end = int(b.starts[r]), int(b.starts[r + 1])
        if start == end:
            continue
        known = min(int(b.totals[r]), b.width * b.page)
        numbers = np.repeat(b.table[r], b.page)[:known]
        seen = np.zeros((known + 1, b.dim))
        there = np.flatnonzero((numbers >= 0) & (numbers < b.pages))
        seen[there + 1, numbers[there] % b.dim] = 1
        seen = np.cumsum(seen, 0)
        at = int(b.totals[r]) - (end - start) + np.arange(end - start)
        counts = seen[np.clip(at + 1, 0, known)] - (seen[np.clip(at + 1 - window, 0, known)] if window else 0)
        want = counts / np.maximum(counts.sum(1, keepdims=True), 1)
        off = np.abs(got[start:end] - want[:, None, :])
        wrong = off > (half + 2.0 ** -21) * want[:, None, :]
        assert not wrong.any(), (r, np.argwhere(wrong)[:4].tolist())


def one_of_each_tile(batch, rows, seed):
    """A token of each 128-row or smaller tile (all heads' at once), the first and the last of each request."""
    rng, step, tokens = np.random.default_rng(seed), max(1, rows * batch.kv_heads // batch.q_heads), set()
    for a, b in zip(batch.starts, batch.starts[1:]):
        tokens |= {int(min(rng.integers(t, t + step), b - 1)) for t in range(a, b, step)} | ({int(a), int(b) - 1} if b > a else set())
    return sorted(tokens)


UNEVEN = [(0, 900), (700, 300), (50, 1), (0, 0), (1300, 500), (3, 1), (2000, 129), (17, 230)]


@pytest.mark.parametrize("dtype,q_heads,kv_heads,dim,page", [("bf16", 16, 2, 64, 16), ("bf16", 16, 4, 128, 64), ("f32", 16, 2, 64, 16), ("f32", 8, 4, 80, 48)])
@pytest.mark.parametrize("window", [0, 300])
def test_equal_shares_cut_tiles(gpu, dtype, q_heads, kv_heads, dim, page, window):
    """More tiles than workgroups: shares that begin and end inside tiles, with whole ones and the next request's between."""
    lengths = UNEVEN if dtype == "bf16" else UNEVEN + [(5, 700)]
    b = Batch(dtype, lengths, q_heads, kv_heads, dim, page, seed=61)
    op = b.op(window=window)
    few, pieces, stopped = deal(b, op, window)
    both = [p for p in pieces if len(p) > 1 and p[0][3] > 0 and p[-1][3] == 0 and p[-1][4] < p[-1][5]]   # ends one tile, begins another
    assert not few and both and any(p[0][0] != p[-1][0] for p in pieces if len(p) > 1)
    assert window or any(len(p) > 2 for p in both)
    assert (stopped > 0) == (window > 0)
    check_tokens(b, b.run(op), one_of_each_tile(b, form_of(op)[0], 61), window)
    check_counts(b, op, window)


class Pool(Batch):
    """Requests of many keys, whose pages are drawn with repetition from few; `holes` columns in a thousand have no page."""

    def __init__(self, dtype, lengths, q_heads, kv_heads, dim, page, pages, seed, holes=0):
        super().__init__(dtype, [(0, 1)], q_heads, kv_heads, dim, page, seed)
        rng = np.random.default_rng(seed)
        self.lengths, self.requests, self.pages = lengths, len(lengths), pages
        self.totals = np.array([c + n for c, n in lengths], np.int32)
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in lengths])]).astype(np.int32)
        self.width, self.tokens = -(-int(self.totals.max()) // page) + 1, int(self.starts[-1]) + 2
        self.table = rng.integers(0, pages, (self.requests, self.width)).astype(np.int32)
        self.table[rng.integers(0, 1000, self.table.shape) < holes] = -1
        for r, total in enumerate(self.totals):
            self.table[r, -(-int(total) // page):] = -1
        self.q, self.q64 = values(dtype, seed, 3, (self.tokens, q_heads, dim), 2.0)
        self.keys, self.values = (values(dtype, seed, i, (pages, page, kv_heads, dim))[0] for i in (4, 5))

    def own_page(self, r, j):
        """Gives key j of request r a page of its own, with the values of one of the others; -> (page, place)."""
        self.keys, self.values = (np.concatenate([x, x[:1]]) for x in (self.keys, self.values))
        self.table[r, j // self.page] = self.pages
        self.pages += 1
        return self.pages - 1, j % self.page


@pytest.mark.parametrize("holes", [0, 30])
@pytest.mark.parametrize("dim", [64, 128])
def test_more_blocks_than_page_numbers_at_once_prompts(gpu, dim, holes):
    """128-row tiles: a half of a piece has more than the 64 blocks whose pages are looked up at a time."""
    b = Pool("bf16", [(44000, 520), (36000, 450), (20, 1)], 8, 1, dim, 16, 700, seed=62, holes=holes)
    op = b.op()
    few, pieces, _ = deal(b, op)
    assert form_of(op)[0] == 128 and not few and sum(p[4] - p[3] > 130 for w in pieces for p in w) > 100
    tokens = one_of_each_tile(b, 128, 62)
    check_tokens(b, b.run(op), tokens[::10] + tokens[-2:])
    check_counts(b, op)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new,group", [(1, 2), (3, 8)])
@pytest.mark.parametrize("dim,holes", [(64, 0), (128, 30), (80, 30)])
def test_more_blocks_than_page_numbers_at_once_tokens(gpu, dtype, new, group, dim, holes):
    """16- and 32-row tiles: a wave has more than the 32 blocks whose pages are looked up at a time."""
    rng = np.random.default_rng(63)
    b = Pool(dtype, [(int(c), new) for c in rng.integers(60000, 80000, 32)], 2 * group, 2, dim, 16, 600, seed=63, holes=holes)
    op = b.op(max_new=new)
    _, pieces, _ = deal(b, op)
    assert form_of(op)[0] == (16 if new * group <= 16 else 32) and sum(p[4] - p[3] > 130 for w in pieces for p in w) > 100
    check_tokens(b, b.run(op), [0, int(b.starts[-1]) - 1])
    check_counts(b, op)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new,group", [(1, 2), (3, 8)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_that_outgrows_the_reference_late(gpu, dtype, new, group, dim):
    """Keys whose scores are more than 2^40 times those before them, past the blocks in which a wave's reference follows its scores: one in a request, three alike in
    pieces of their own, and, of new tokens, ones that some of a tile's rows do not see."""
    rng = np.random.default_rng(64)
    b = Pool(dtype, [(int(c), new) for c in rng.integers(25000, 30000, 80)], group, 1, dim, 16, 600, seed=64)
    op = b.op(max_new=new)
    _, pieces, _ = deal(b, op)
    block, late = form_of(op)[1], 0

    def places(r):   # keys 20 blocks behind the begin of pieces of a request
        return [(b0 + 20) * block + 5 for w in pieces for (q, _, _, b0, b1, _) in w if q == r and b1 - b0 > 24]

    total = b.totals
    planted = {0: places(0)[-1:], 25: places(25)[:3], 50: [int(total[50]) - 1], 75: places(75)[:1] + [int(total[75]) - (2 if new > 1 else 1)]}
    assert len(places(25)) >= 3 and all(planted.values())
    for r, keys in planted.items():
        token = int(b.starts[r + 1]) - 1
        for j in keys:
            page, place = b.own_page(r, j)
            q = b.q64[token, 0]   # (the last new token's first query head)
            k = q * (90 * dim ** 0.5 / (q @ q))   # a score of 90; the others' are within 20
            b.keys[page, place, 0] = M.synth.f32_to_bf16_bits(k.astype(np.float32)) if dtype == "bf16" else k.astype(np.float32)
            late += sum(b0 + 16 < j // block < b1 for w in pieces for (of, _, _, b0, b1, _) in w if of == r)
    assert late >= 5, late
    tokens = sorted({int(t) for r in planted for t in (b.starts[r], b.starts[r + 1] - 1)} | ({int(b.starts[75]) + 1} if new > 1 else set()))
    check_tokens(b, b.run(b.op(max_new=new)), tokens)   # (an op with the pages that came)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [0, 40, 5000])
def test_more_new_tokens_than_the_table_holds(gpu, dtype, window):
    """Keys past the table are hidden; the tiles there have no more blocks than the table."""
    b = Batch(dtype, [(0, 2500), (600, 3000), (3, 1), (100, 700)], 8, 2, 64, 16, seed=65)
    b.width, b.table = 40, b.table[:, :40].copy()
    b.keys[...], b.values[...] = (np.where(x == x, x, 0) if dtype == "f32" else np.where((x & 0x7fff) > 0x7f80, 0, x) for x in (b.keys, b.values))
    op = b.op(window=window)
    few, pieces, stopped = deal(b, op, window)
    assert not few and stopped > 50 and max(p[5] for w in pieces for p in w) <= 40 * 16 // form_of(op)[1]
    check_tokens(b, b.run(op), one_of_each_tile(b, 128, 65)[::2], window)
    check_counts(b, op, window)
