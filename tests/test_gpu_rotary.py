"""Rotary positions against the formula in 64 bits, the gradient against differences, keys and values in their slots."""
import numpy as np
import pytest

import morello_amd as M
from paged_util import DTYPE, HALF_STEP, STORED, as_f64, values

pytestmark = pytest.mark.gpu


def turned(x, positions, frequencies, sections, adjacent, inverse=False):
    """(result, bound) in 64 bits.  The sine and cosine of an angle are off by at most 2^-23 (the angle's own rounding in 64 bits: below 2^31 * 2^-52
    turns), two products and a sum round by half a step of 32 bits each, and the result is rounded once."""
    pairs = sum(sections)
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = positions[axis].T.astype(np.float64) * frequencies.astype(np.float64) * (-1 if inverse else 1)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    lo, hi = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    y, size = x.copy(), np.zeros_like(x)
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    size[..., lo] = size[..., hi] = np.abs(x[..., lo]) + np.abs(x[..., hi])
    return y, size


def bound(y, size, dtype):
    return np.where(size > 0, HALF_STEP[dtype] * np.abs(y), 0) + (1 + HALF_STEP[dtype]) * size * (2.0 ** -23 + 2 * 2.0 ** -24)


def strided(stored, strides, fill):
    """A buffer that holds `stored` [tokens][heads][dim] at these strides, `fill` between."""
    t, h, d = stored.shape
    flat = np.full((t - 1) * strides[0] + (h - 1) * strides[1] + d, fill, stored.dtype)
    view = np.lib.stride_tricks.as_strided(flat, stored.shape, (strides[0] * stored.itemsize, strides[1] * stored.itemsize, stored.itemsize))
    view[...] = stored
    return flat, view


def run(op, arrays):
    bufs = [M.DeviceBuffer.from_numpy(a) if a is not None else None for a in arrays]
    op.run_device([b.ptr if b else None for b in bufs])
    got = [b.to_numpy(a.dtype, a.shape) if b else None for a, b in zip(arrays, bufs)]
    for b in bufs:
        if b:
            b.free()
    return got


def positions_of(seed, axes, tokens, far):
    return np.random.default_rng(seed).integers(0, far, (axes, tokens)).astype(np.int32)


def frequencies_of(pairs):
    return (10000.0 ** (-np.arange(pairs) / pairs)).astype(np.float32)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,sections,page,far", [
    (1, 4, 1, 64, [32], 16, 100), (37, 8, 2, 128, [16, 24, 24], 16, 5000), (70, 3, 3, 80, [20], 64, 2 ** 31 - 1), (33, 5, 1, 96, [1, 2, 3, 4], 7, 10 ** 6),
    (5, 2, 2, 7, [3], 1, 4096), (129, 1, 1, 256, [128], 32, 10 ** 5), (3, 2, 1, 1024, [500, 12], 5, 3), (2, 48, 8, 128, [64], 16, 10)])
def test_into_pages(gpu, dtype, adjacent, tokens, q_heads, kv_heads, dim, sections, page, far):
    """A slot of every third token lies outside the cache: its keys and values are left out, its queries are turned."""
    q, q64 = values(dtype, 1, 0, (tokens, q_heads, dim))
    k, k64 = values(dtype, 1, 1, (tokens, kv_heads, dim))
    v, v64 = values(dtype, 1, 2, (tokens, kv_heads, dim))
    pos, freq = positions_of(2, len(sections), tokens, far), frequencies_of(sum(sections))
    pages = -(-tokens // page) + 2
    slots = np.random.default_rng(4).permutation(pages * page)[:tokens].astype(np.int32)
    slots[2::3] = np.resize([-1, pages * page, -2 ** 31, 2 ** 31 - 1], len(slots[2::3]))
    kept = (slots >= 0) & (slots < pages * page)
    op = M.Rotary(DTYPE[dtype], tokens, q_heads, kv_heads, dim, sections, adjacent, page_size=page, pages=pages)
    old = values(dtype, 1, 3, (pages * page, kv_heads, dim))[0]
    got = run(op, [q, k, v, pos, freq, slots, np.zeros_like(q), old.copy(), old.copy()])
    y, size = turned(q64, pos, freq, sections, adjacent)
    assert (np.abs(as_f64(dtype, got[6]) - y) <= bound(y, size, dtype)).all()
    y, size = turned(k64, pos, freq, sections, adjacent)
    assert (np.abs(as_f64(dtype, got[7][slots[kept]]) - y[kept]) <= bound(y, size, dtype)[kept]).all()
    assert np.array_equal(got[8][slots[kept]], v[kept])
    rest = np.setdiff1d(np.arange(pages * page), slots[kept])
    assert np.array_equal(got[7][rest], old[rest]) and np.array_equal(got[8][rest], old[rest])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("odd", [0, 1])
def test_strides_and_in_place(gpu, dtype, adjacent, odd):
    """Queries and keys that lie in one row of all projections, whole chunks apart or not, turned where they are; what lies between stays."""
    tokens, q_heads, kv_heads, dim, sections = 50, 6, 2, 64, [8, 16]
    row = (q_heads + 2 * kv_heads) * dim + odd
    qkv, qkv64 = values(dtype, 5, 0, (tokens, row))
    pos, freq = positions_of(6, 2, tokens, 3000), frequencies_of(24)
    strides = (row, dim)
    op = M.Rotary(DTYPE[dtype], tokens, q_heads, kv_heads, dim, sections, adjacent, q_strides=strides, k_strides=strides, q_out_strides=strides,
                  key_strides=(0, row, dim))
    buf = M.DeviceBuffer.from_numpy(qkv)
    rest = [M.DeviceBuffer.from_numpy(a) for a in (pos, freq)]
    k = buf.ptr + q_heads * dim * qkv.itemsize
    op.run_device([buf.ptr, k, None, rest[0].ptr, rest[1].ptr, None, buf.ptr, k, None])
    got = buf.to_numpy(qkv.dtype, qkv.shape)
    heads = qkv64[:, :(q_heads + kv_heads) * dim].reshape(tokens, -1, dim)
    y, size = turned(heads, pos, freq, sections, adjacent)
    g = as_f64(dtype, got[:, :(q_heads + kv_heads) * dim]).reshape(heads.shape)
    assert (np.abs(g - y) <= bound(y, size, dtype)).all()
    assert np.array_equal(got[:, (q_heads + kv_heads) * dim:], qkv[:, (q_heads + kv_heads) * dim:])
    # into others, heads first
    out = np.zeros((q_heads, tokens, dim), STORED[dtype])
    keys = np.zeros((kv_heads, tokens, dim), STORED[dtype])
    op = M.Rotary(DTYPE[dtype], tokens, q_heads, kv_heads, dim, sections, adjacent, q_strides=strides, k_strides=strides,
                  q_out_strides=(dim, tokens * dim), key_strides=(0, dim, tokens * dim))
    bufs = [M.DeviceBuffer.from_numpy(a) for a in (qkv, out, keys)]
    op.run_device([bufs[0].ptr, bufs[0].ptr + q_heads * dim * qkv.itemsize, None, rest[0].ptr, rest[1].ptr, None, bufs[1].ptr, bufs[2].ptr, None])
    again = np.concatenate([bufs[1].to_numpy(out.dtype, out.shape), bufs[2].to_numpy(keys.dtype, keys.shape)]).transpose(1, 0, 2)
    assert np.array_equal(again.reshape(tokens, -1), got[:, :(q_heads + kv_heads) * dim])


def test_queries_alone(gpu):
    q, q64 = values("bf16", 7, 0, (9, 4, 32))
    pos, freq = positions_of(8, 1, 9, 77), frequencies_of(16)
    got = run(M.Rotary(M.bf16, 9, 4, 0, 32, [16]), [q, None, None, pos, freq, None, np.zeros_like(q), None, None])[6]
    y, size = turned(q64, pos, freq, [16], False)
    assert (np.abs(as_f64("bf16", got) - y) <= bound(y, size, "bf16")).all()


@pytest.mark.parametrize("adjacent", [False, True])
def test_inverse_is_the_gradient(gpu, adjacent):
    """<g, R(x + e) - R(x - e)> / 2 = <inverse(g), e> for a linear R, and the inverse undoes the rotation."""
    tokens, heads, dim, sections = 21, 3, 48, [5, 9]
    x, x64 = values("f32", 9, 0, (tokens, heads, dim))
    g, g64 = values("f32", 9, 1, (tokens, heads, dim))
    e, e64 = values("f32", 9, 2, (tokens, heads, dim))
    pos, freq = positions_of(10, 2, tokens, 100000), frequencies_of(14)

    def call(a, inverse):
        op = M.Rotary(M.f32, tokens, heads, heads, dim, sections, adjacent, inverse)
        got = run(op, [a, a, None, pos, freq, None, np.zeros_like(a), np.zeros_like(a), None])
        assert np.array_equal(got[6], got[7])
        return got[6].astype(np.float64)

    gradient = call(g, True)
    y, size = turned(g64, pos, freq, sections, adjacent, True)
    assert (np.abs(gradient - y) <= bound(y, size, "f32")).all()
    plus, minus = (x64 + e64).astype(np.float32), (x64 - e64).astype(np.float32)
    difference = float((g64 * (call(plus, False) - call(minus, False))).sum() / 2)
    # every one of the sums' terms is off by at most 8 half steps of |g| (|x| + |e|) of its pair, and a step of the inputs' own rounding
    slack = 16 * 2.0 ** -24 * float((np.abs(g64) * (np.abs(x64) + np.abs(e64) + 2)).sum()) * 2
    assert abs(difference - float((gradient * e64).sum())) <= slack
    back = call(call(x, False).astype(np.float32), True)
    assert np.abs(back - x64).max() <= 8 * 2.0 ** -23 * (np.abs(x64).max() * 2)


def test_refused_pointers(gpu):
    op = M.Rotary(M.bf16, 2, 1, 1, 8, [4], page_size=4, pages=2)
    buf = M.DeviceBuffer(4096)
    for i in range(9):
        with pytest.raises(M.MorelloError) as err:
            op.run_device([None if j == i else buf.ptr + 256 * j for j in range(9)])
        assert err.value.status == 6
    op = M.Rotary(M.bf16, 2, 2, 1, 8, [4], q_out_strides=(32, 8))
    with pytest.raises(M.MorelloError) as err:
        op.run_device([buf.ptr, buf.ptr + 1024, None, buf.ptr + 2048, buf.ptr + 2304, None, buf.ptr, buf.ptr + 1024, None])
    assert err.value.status == 3 and "other strides" in str(err.value)
