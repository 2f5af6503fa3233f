"""Attention over pages against the formula in 64 bits; every slot without a key of its request, and every row without a token, holds NaN."""
import numpy as np
import pytest

import morello_amd as M
from paged_util import POISON, Batch, as_f64

pytestmark = pytest.mark.gpu

DECODE = [(0, 1), (1, 1), (15, 1), (16, 1), (300, 1), (31, 1), (32, 1), (63, 1), (511, 1), (90, 1)]
CHUNKS = [(0, 1), (0, 40), (100, 17), (33, 1), (0, 0), (64, 64), (5, 130), (250, 1), (7, 0), (1, 33)]


def run_and_check(batch, window=0, scale=None, **given):
    if scale is not None:
        given["scale"] = scale
    got = batch.run(batch.op(window=window, **given))
    batch.check(got, window, scale)
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(1, 1), (4, 1), (8, 2), (6, 2), (3, 3), (16, 1)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_heads(gpu, dtype, heads, dim, lengths):
    run_and_check(Batch(dtype, lengths, *heads, dim, 16, seed=11))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [8, 32, 40, 80, 96, 120, 200, 20, 3])
def test_head_dims(gpu, dtype, dim):
    run_and_check(Batch(dtype, DECODE[:6] + CHUNKS[:6], 4, 2, dim, 32, seed=12))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 48, 64, 128, 1000])
@pytest.mark.parametrize("heads_first", [False, True])
def test_page_sizes(gpu, dtype, page, heads_first):
    run_and_check(Batch(dtype, [(0, 1), (100, 1), (70, 30), (129, 3), (0, 70)], 4, 2, 64, page, seed=13, heads_first=heads_first))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 100, 5000])
def test_windows(gpu, dtype, window):
    run_and_check(Batch(dtype, [(0, 1), (300, 1), (129, 1), (0, 100), (200, 70), (70, 3)], 4, 1, 64, 16, seed=14), window=window)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_long_and_short_contexts_together(gpu, dtype):
    """One request's keys shared out over many workgroups, others of a block or none."""
    run_and_check(Batch(dtype, [(6000, 1), (3, 1), (0, 1), (2047, 1)], 4, 2, 128, 64, seed=15))
    run_and_check(Batch(dtype, [(4000, 1)], 8, 1, 64, 16, seed=16))
    run_and_check(Batch(dtype, [(2500, 20), (3, 1), (900, 1)], 4, 1, 64, 32, seed=17))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_requests(gpu, dtype):
    rng = np.random.default_rng(1)
    lengths = [(int(c), int(n)) for c, n in zip(rng.integers(0, 30, 700), rng.choice([0, 1, 1, 1, 2], 700))]
    run_and_check(Batch(dtype, lengths, 2, 1, 32, 16, seed=18))
    run_and_check(Batch(dtype, [(c, min(n, 1)) for c, n in lengths], 2, 2, 64, 16, seed=19))


def widened(batch, keys):
    """With a table that has room for so many keys of a request: small tables and large ones are dealt to workgroups in ways of their own."""
    width = -(-keys // batch.page)
    batch.table = np.pad(batch.table, ((0, 0), (0, width - batch.width)), constant_values=-1)
    batch.width = width
    return batch


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,dim", [((4, 1), 64), ((6, 2), 128), ((3, 3), 80), ((16, 1), 96)])
@pytest.mark.parametrize("lengths", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_wide_tables(gpu, dtype, heads, dim, lengths):
    run_and_check(widened(Batch(dtype, lengths, *heads, dim, 16, seed=51), 5000))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_requests_in_wide_tables(gpu, dtype):
    rng = np.random.default_rng(2)
    lengths = [(int(c), int(n)) for c, n in zip(rng.integers(0, 30, 700), rng.choice([0, 1, 1, 1, 2], 700))]
    run_and_check(widened(Batch(dtype, lengths, 2, 1, 32, 16, seed=52), 2000))
    run_and_check(widened(Batch(dtype, [(c, min(n, 1)) for c, n in lengths], 2, 2, 64, 16, seed=53), 2000))
    lengths = [(int(c), int(n)) for c, n in zip(rng.integers(0, 300, 130), rng.choice([0, 0, 0, 1, 40], 130))]
    run_and_check(widened(Batch(dtype, lengths, 4, 2, 64, 16, seed=54), 2000), window=100)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("keys", [400, 3000])
def test_more_new_tokens_than_the_bound_says(gpu, dtype, keys):
    """max_new is taken at its word for choosing kernels only: requests of more tokens have more tiles than one."""
    run_and_check(widened(Batch(dtype, [(0, 1), (100, 70), (17, 33), (0, 0), (250, 2)], 4, 2, 64, 16, seed=55), keys), max_new=1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_queries_far_apart(gpu, dtype):
    """Tokens whose queries lie 8 MB and more apart: past what one resource over a tile's queries would hold."""
    b = widened(Batch(dtype, [(0, 20), (90, 3)], 2, 1, 64, 16, seed=56, spare_rows=0), 2000)
    stride, size = 1 << 22, b.q.itemsize
    q = M.DeviceBuffer(((b.tokens - 1) * stride + b.q_heads * b.dim) * size)
    for t in range(b.tokens):
        row = np.ascontiguousarray(b.q[t])
        M._check(M.B.load().mrl_memcpy_h2d(q.ptr + t * stride * size, row.ctypes.data, row.nbytes), "mrl_memcpy_h2d")
    op = b.op(max_new=20, q_strides=(stride, b.dim))
    out = np.full((b.tokens, b.q_heads, b.dim), 5, np.float32).astype(b.q.dtype) if dtype == "f32" else np.full((b.tokens, b.q_heads, b.dim), 0x40a0, np.uint16)
    bufs = [M.DeviceBuffer.from_numpy(a) for a in (b.keys, b.values, b.table, b.starts, b.totals, out, np.full(max(16, op.workspace_bytes()), 0xff, np.uint8))]
    op.run_device([q.ptr] + [x.ptr for x in bufs])
    b.check(bufs[5].to_numpy(out.dtype, out.shape))
    for x in bufs + [q]:
        x.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_that_see_nothing(gpu, dtype):
    """Lengths below the new tokens, of zero and below; tables whose numbers lie outside the cache, or which end before the length: zeros where
    no key is left."""
    for lengths in ([(40, 1), (70, 1), (50, 1)], [(40, 5), (70, 20), (0, 40)]):
        b = Batch(dtype, lengths, 4, 2, 64, 16, seed=20)
        b.totals[:] = [0, lengths[1][0] + lengths[1][1], -7 if lengths[2][1] == 1 else 13]
        b.table[1, [0, 2]] = [-1, b.pages]
        got = as_f64(dtype, run_and_check(b))
        assert (got[b.starts[0]:b.starts[1]] == 0).all()
        b = Batch(dtype, lengths, 4, 2, 64, 16, seed=21)
        b.table[:] = [[-1], [2 ** 31 - 1], [-2 ** 31]]
        assert (as_f64(dtype, run_and_check(b))[b.starts[0]:b.starts[3]] == 0).all()
        b = Batch(dtype, lengths, 4, 2, 64, 16, seed=22)
        b.totals[:] += 3 * b.width * 16   # past the table: what it holds is seen by every token
        b.keys[...], b.values[...] = (np.where(x == x, x, 0) if dtype == "f32" else np.where((x & 0x7fff) > 0x7f80, 0, x) for x in (b.keys, b.values))
        b.table[b.table < 0] = 0
        run_and_check(b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [0, 20])
def test_poison_in_masked_places(gpu, dtype, window):
    """NaN and infinity in the keys and values of tokens behind a row's own (and, with a window, before it) reach only the rows that see them."""
    b = Batch(dtype, [(50, 60), (33, 100), (200, 1)], 4, 2, 64, 16, seed=23)
    want, bound = b.want(window)
    hurt = np.zeros(b.tokens, bool)
    inf = {"bf16": np.uint16(0x7f80), "f32": np.float32(np.inf)}[dtype]
    for r, j in ((0, 80), (1, 70), (1, 101)):
        page, place = b.table[r, j // 16], j % 16
        b.keys[page, place, 0], b.values[page, place, 0] = POISON[dtype], POISON[dtype]
        b.values[page, place, 1] = inf
        first = int(b.starts[r + 1]) - (int(b.totals[r]) - j)
        hurt[first:int(b.starts[r + 1]) if not window else min(first + window, int(b.starts[r + 1]))] = True
    got = as_f64(dtype, b.run(b.op(window=window)))
    end = int(b.starts[-1])
    fine = ~hurt[:end]
    off = np.abs(got[:end] - want[:end])[fine]
    assert np.isfinite(got[:end][fine]).all() and (off <= bound[:end][fine]).all()
    assert np.isnan(got[:end, :2][hurt[:end]]).all() and not np.isfinite(got[:end, 2:][hurt[:end]]).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scores_far_apart(gpu, dtype):
    """Scores of a standard deviation of 60, a negative scale, one key that outweighs the rest late in the cache, and scores of -infinity."""
    for lengths in ([(700, 1), (90, 1)], [(300, 150), (90, 40)]):
        run_and_check(Batch(dtype, lengths, 4, 1, 64, 16, seed=24, q_std=60.0))
        run_and_check(Batch(dtype, lengths, 4, 1, 64, 16, seed=25), scale=-0.3)
        b = Batch(dtype, lengths, 4, 1, 64, 16, seed=26)
        b.q[..., 0] = {"bf16": np.uint16(0x3f80), "f32": np.float32(1)}[dtype]
        b.q64[..., 0] = 1
        for r in range(2):
            for j in range(5, sum(lengths[r]), 9):
                b.keys[b.table[r, j // 16], j % 16, 0, 0] = {"bf16": np.uint16(0xff80), "f32": np.float32(-np.inf)}[dtype]
        run_and_check(b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_strides_and_alignment(gpu, dtype, lengths):
    """q as a part of a row of all projections, out heads first, values between other things; then the same on odd strides and addresses."""
    b = Batch(dtype, lengths, 4, 2, 64, 16, seed=27)
    plain = run_and_check(b)
    for row, shift in ((4 * 64 + 256, 0), (4 * 64 + 3, 1)):
        item = b.q.itemsize
        q = np.full((b.tokens, row), POISON[dtype], b.q.dtype)
        q[:, :256] = b.q.reshape(b.tokens, -1)
        cache = np.full((b.pages, 16, 2, 2, 64 + shift), POISON[dtype], b.q.dtype)   # keys and values of a head beside each other
        cache[:, :, :, 0, :64], cache[:, :, :, 1, :64] = b.keys, b.values
        strides = (16 * 4 * (64 + shift), 4 * (64 + shift), 2 * (64 + shift))
        out = np.full((4, b.tokens, 64 + shift), {"bf16": np.uint16(0x40a0), "f32": np.float32(5)}[dtype], b.q.dtype)
        op = b.op(q_strides=(row, 64), key_strides=strides, value_strides=strides, out_strides=(64 + shift, b.tokens * (64 + shift)))
        bufs = [M.DeviceBuffer.from_numpy(a) for a in (q, cache, b.table, b.starts, b.totals, out)] + [M.DeviceBuffer(max(16, op.workspace_bytes()))]
        at = [x.ptr for x in bufs]
        op.run_device([at[0], at[1], at[1] + (64 + shift) * item, at[2], at[3], at[4], at[5], at[6]])
        got = bufs[5].to_numpy(out.dtype, out.shape)
        assert np.array_equal(got[:, :, 64:], out[:, :, 64:])
        got = got[:, :, :64].transpose(1, 0, 2)
        b.check(got)
        if not shift:
            assert np.array_equal(got, plain)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_bound_of_new_tokens_chooses_kernels_only(gpu, dtype):
    """Results are right whatever the bound says, too low ones too."""
    b = Batch(dtype, CHUNKS, 4, 2, 64, 16, seed=28)
    for most in (0, 1, 5, 8, 40, 10 ** 6):
        run_and_check(b, max_new=most)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_first_rows_of_no_request_and_starts_past_the_rows(gpu, dtype):
    b = Batch(dtype, [(20, 3), (50, 1), (9, 30)], 4, 2, 64, 16, seed=29, first=7)
    run_and_check(b)
    # starts past `tokens`: the rows that there are, nothing behind them
    for lengths in ([(20, 1), (50, 1)], [(20, 3), (50, 40)]):
        b = Batch(dtype, lengths, 4, 2, 64, 16, seed=30, spare_rows=0)
        want = b.run(b.op())
        starts = b.starts.copy()
        b.starts = np.array([starts[0], starts[1], 10 ** 6], np.int32)
        got = b.run(b.op())
        assert np.array_equal(got[:starts[1]], want[:starts[1]]) and np.isfinite(as_f64(dtype, got)).all()


def test_caches_past_4_gib(gpu):
    """Pages whose elements lie past 2^31 and 2^32 bytes of the cache: one request whose few keys are in the last pages."""
    free = M.device_free_bytes()
    if free < 40 << 30:
        pytest.skip("needs 20 GiB of device memory")
    page, kv, dim, pages = 64, 8, 128, 40000   # 5.2 GB each of keys and values
    small = Batch("bf16", [(150, 1), (70, 40)], 16, kv, dim, page, seed=31)
    op = small.op(pages=pages)
    where = np.array([pages - 1, 16383, 16384, 32767, 32768, 5, pages - 2, 39000, 8191, 8192][:small.pages], np.int32)
    bytes_ = page * kv * dim * 2
    caches = [M.DeviceBuffer(pages * bytes_) for _ in range(2)]
    for cache, host in zip(caches, (small.keys, small.values)):
        for i, p in enumerate(where):
            one = np.ascontiguousarray(host[i])
            M._check(M.B.load().mrl_memcpy_h2d(cache.ptr + int(p) * bytes_, one.ctypes.data, one.nbytes), "mrl_memcpy_h2d")
    table = np.where(small.table >= 0, where[np.maximum(small.table, 0)], -1).astype(np.int32)
    out = np.full((small.tokens, 16, dim), 0x40a0, np.uint16)
    bufs = [M.DeviceBuffer.from_numpy(a) for a in (small.q, table, small.starts, small.totals, out)] + [M.DeviceBuffer(max(16, op.workspace_bytes()))]
    op.run_device([bufs[0].ptr, caches[0].ptr, caches[1].ptr, bufs[1].ptr, bufs[2].ptr, bufs[3].ptr, bufs[4].ptr, bufs[5].ptr])
    got = bufs[4].to_numpy(out.dtype, out.shape)
    for x in caches + bufs:
        x.free()
    small.check(got)


def test_refused_pointers(gpu):
    b = Batch("bf16", [(20, 1)], 4, 2, 64, 16, seed=32)
    op = b.op()
    buf = M.DeviceBuffer(1 << 20)
    for i in range(7):
        with pytest.raises(M.MorelloError) as err:
            op.run_device([None if j == i else buf.ptr + 4096 * j for j in range(8)])
        assert err.value.status == 6
    with pytest.raises(M.MorelloError) as err:
        op.run_device([buf.ptr + 4096 * j + (8 if j == 7 else 0) for j in range(8)])
    assert err.value.status == 1 and "workspace" in str(err.value)
