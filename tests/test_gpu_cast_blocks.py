"""Casts to e4m3 with a scale for each block: bit for bit where nothing but divisions, products and roundings in 32 bits is done, within half a step behind a gate."""
import numpy as np
import pytest

import morello_amd as M
from blocks_util import DTYPE, E4M3, POISON, U, Device, as_f64, back, cast, over_blocks, strided, values

pytestmark = pytest.mark.gpu


def run(dtype, x, rows, cols, high, gated=False, x_stride=0, out_stride=0, scale_stride=0, x_offset=0, out_offset=0):
    """x: stored values -> (bytes, scales); what lies between rows is checked to be as it was."""
    blocks, highs = -(-cols // 128), -(-rows // high)
    x_flat, _ = strided(x, x_stride or x.shape[1], POISON[dtype], x_offset)
    out_flat, _ = strided(np.full((rows, cols), 0x5a, np.uint8), out_stride or cols, 0xa5, out_offset)
    scale_flat, _ = strided(np.full((highs, blocks), 5, np.float32), scale_stride or blocks, 9)
    op = M.CastBlocks(DTYPE[dtype], rows, cols, high, gated, x_stride, out_stride, scale_stride)
    with Device() as d:
        op.run_device([d.put(x_flat, x_offset), d.put(out_flat, out_offset), d.put(scale_flat)])
        out, scales = d.get(1, out_flat), d.get(2, scale_flat)
    view = lambda flat, offset, shape, stride: np.lib.stride_tricks.as_strided(flat[offset:], shape, (stride * flat.itemsize, flat.itemsize))
    got = view(out, out_offset, (rows, cols), out_stride or cols).copy(), view(scales, 0, (highs, blocks), scale_stride or blocks).copy()
    view(out, out_offset, (rows, cols), out_stride or cols)[:] = 0x5a
    view(scales, 0, (highs, blocks), scale_stride or blocks)[:] = 5
    assert np.array_equal(out, out_flat) and np.array_equal(scales, scale_flat), "written between the rows"
    return got


def same(got, want):
    assert np.array_equal(got[1].view(np.uint32), want[1].view(np.uint32)), "scales"
    nan = np.isnan(E4M3[want[0]])
    assert np.array_equal(np.isnan(E4M3[got[0]]), nan) and np.array_equal(got[0][~nan], want[0][~nan])


SIZES = [(1, 1), (1, 128), (3, 127), (16, 4096), (5, 1000), (129, 130), (128, 128), (300, 513), (2, 8)]


@pytest.mark.parametrize("high", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_bytes_and_scales(gpu, dtype, high, rows, cols):
    x, x64 = values(dtype, rows + cols, 0, (rows, cols), 3.0)
    same(run(dtype, x, rows, cols, high), cast(x64, high))


@pytest.mark.parametrize("high", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_and_odd_addresses(gpu, dtype, high):
    rows, cols = 131, 261
    x, x64 = values(dtype, 7, 0, (rows, cols))
    want = cast(x64, high)
    for kw in (dict(x_stride=300, out_stride=272, scale_stride=8), dict(x_stride=263, x_offset=3, out_stride=267, out_offset=5, scale_stride=3)):
        same(run(dtype, x, rows, cols, high, **kw), want)


@pytest.mark.parametrize("high", [1, 128])
def test_blocks_of_nothing_tiny_and_unbounded_values(gpu, high):
    rows, cols = 256, 640
    x = values("f32", 8, 0, (rows, cols))[0].copy()
    x[:128, :128] = 0
    x[:128, 128:256] = np.float32(1e-44) * np.sign(x[:128, 128:256])
    x[:128, 256:384] *= np.float32(2.0 ** -112)
    x[:, 384:512] *= np.float32(1e37)
    x[5, 3], x[130, 200], x[200, 600] = np.nan, np.inf, -np.inf
    x[140, 256:384] = np.nan
    x[0, 512:640] = np.where(np.arange(128) % 2, 448, np.arange(128) * 0.5)   # sums that lie between two numbers
    got, want = run("f32", x, rows, cols, high), cast(x, high)
    same(got, want)
    with np.errstate(invalid="ignore"):
        read = back(got[0], got[1], high)
    assert not read[:128, :128][~np.isnan(x[:128, :128])].any() and np.isnan(read[5, 3]) and np.isnan(read[130, 128:256]).all()


def test_every_number_of_the_type_and_those_between(gpu):
    """With a largest value of 448 the scale is 1: all numbers of e4m3, all that lie halfway, and their neighbours in f32."""
    grid = np.sort(E4M3[:127]).astype(np.float32)
    half = ((grid[1:].astype(np.float64) + grid[:-1]) / 2).astype(np.float32)
    every = np.concatenate([grid, half, np.nextafter(half, np.float32(0)), np.nextafter(half, np.float32(500))])
    every = np.concatenate([every, -every])
    x = np.zeros((-(-len(every) // 127), 128), np.float32)
    x[:, 127] = 448
    for i, v in enumerate(every):
        x[i // 127, i % 127] = v
    got = run("f32", x, *x.shape, 1)
    assert (got[1] == 1).all()
    same(got, cast(x, 1))


@pytest.mark.parametrize("high", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (4, 128), (33, 300), (130, 1001)])
def test_behind_a_gate(gpu, dtype, high, rows, cols):
    """silu takes an exponential (good to 2 steps), a sum, a quotient and a product: 8 u in all; then a scale of u more, and half a step of e4m3."""
    x, x64 = values(dtype, rows, 1, (rows, 2 * cols), 4.0)
    bytes_, scales = run(dtype, x, rows, cols, high, gated=True, x_stride=2 * cols + 1)
    g, u = x64[:, :cols], x64[:, cols:]
    y = g / (1 + np.exp(-g)) * u
    want = cast(y, high)
    assert (np.abs(scales / want[1] - 1) <= 10 * U).all()
    read, s = back(bytes_, scales, high), over_blocks(scales.astype(np.float64), rows, cols, high)
    step = np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10)   # half a step, of numbers and below the smallest normal one
    assert (np.abs(read - y) <= step * (1 + 2.0 ** -10) + 16 * U * np.abs(y)).all()


def test_a_gate_far_out(gpu):
    """exp(-g) past 32 bits: silu is 0 there."""
    x = np.array([[-1000, -90, 1000, 0] + [2, 3, 4, 5]], np.float32)
    bytes_, scales = run("f32", x, 1, 4, 1, gated=True)
    assert (np.abs(back(bytes_, scales, 1)[0, [0, 1, 3]]) <= 1e-30).all() and abs(back(bytes_, scales, 1)[0, 2] / 4000 - 1) < 1e-5
    assert (as_f64("f32", scales) > 0).all()
