"""Tensors past 2^32 bytes: rows, experts and results that only 64-bit offsets find."""
import numpy as np
import pytest

import morello_amd as M
from blocks_util import HALF_STEP, Layer, as_f64, back, cast, product_bound, values
from morello_amd import _binding as B
from morello_amd import synth

pytestmark = pytest.mark.gpu


class Space:
    """Device memory of which only some is written and read."""

    def __init__(self, *sizes):
        self.buffers = [M.DeviceBuffer(int(n)) for n in sizes]

    def __enter__(self):
        return self

    def __exit__(self, *_):
        for b in self.buffers:
            b.free()

    def put(self, i, at, x):
        x = np.ascontiguousarray(x)
        assert at + x.nbytes <= self.buffers[i].nbytes
        M._check(B.load().mrl_memcpy_h2d(self.buffers[i].ptr + at, x.ctypes.data, x.nbytes), "mrl_memcpy_h2d")

    def get(self, i, at, like):
        got = np.empty_like(like)
        assert at + got.nbytes <= self.buffers[i].nbytes
        M._check(B.load().mrl_memcpy_d2h(got.ctypes.data, self.buffers[i].ptr + at, got.nbytes), "mrl_memcpy_d2h")
        return got

    def ptr(self, i):
        return self.buffers[i].ptr


@pytest.mark.parametrize("high", [1, 128])
def test_cast_of_rows_far_apart(gpu, high):
    rows, cols, stride, out_stride = 3, 300, 1100000000, 2200000001
    x, x64 = values("bf16", 1, 0, (rows, cols))
    with Space(2 * (2 * stride + cols), 2 * out_stride + cols, 4096) as s:
        for r in range(rows):
            s.put(0, 2 * r * stride, x[r])
        M.CastBlocks(M.bf16, rows, cols, high, x_stride=stride, out_stride=out_stride).run_device([s.ptr(i) for i in range(3)])
        want, scales = cast(x64, high)
        assert np.array_equal(s.get(2, 0, scales.astype(np.float32)), scales.astype(np.float32))
        for r in range(rows):
            assert np.array_equal(s.get(1, r * out_stride, want[r]), want[r])


@pytest.mark.parametrize("m,n,out", [(70000, 33000, "bf16"), (40000, 28000, "f32")])
def test_product_of_many_rows_and_columns(gpu, m, n, out):
    """Checked at the corners and in a row beyond 2^32 bytes."""
    k, size = 256, 2 if out == "bf16" else 4
    (a, a_s), (b, b_s) = cast(synth.normal_f32(2, 0, (512, k)).astype(np.float32), 1), cast(synth.normal_f32(2, 1, (512, k)).astype(np.float32), 128)
    rows, cols = np.arange(m) % 509, np.arange(n) % 512
    with Space(m * k, m * 8, n * k, -(-n // 128) * 8, m * n * size, 16) as s:
        for i, x in enumerate((a[rows], a_s[rows].astype(np.float32), b[cols], b_s[np.arange(-(-n // 128)) % 4].astype(np.float32))):
            s.put(i, 0, x)
        op = M.MatmulBlocks(M.bf16 if out == "bf16" else M.f32, m, n, k)
        assert op.workspace_bytes() <= 16
        op.run_device([s.ptr(i) for i in range(6)])
        a64, b64 = back(a, a_s, 1), back(b, b_s, 128)
        for row in (0, 1, 2 ** 32 // (n * size) + 3, m - 1):
            got = as_f64(out, s.get(4, row * n * size, np.empty(n, np.uint16 if out == "bf16" else np.float32)))
            x = a64[row % 509][None]
            want = (x @ b64.T)[0]
            bound = product_bound(x, b64, 2, HALF_STEP[out], want[None], cut=out == "bf16")[0]
            assert (np.abs(got - want[cols]) <= bound[cols]).all(), row


@pytest.mark.parametrize("m", [2, 40, 130])
def test_product_of_rows_far_apart(gpu, m):
    n, k, stride, scale_stride, out_stride = 70, 300, 2200000032 // (m - 1) // 16 * 16, 640000000 // (m - 1), 1200000000 // (m - 1)
    (a, a_s), (b, b_s) = cast(synth.normal_f32(3, 0, (m, k)).astype(np.float32), 1), cast(synth.normal_f32(3, 1, (n, k)).astype(np.float32), 128)
    op = M.MatmulBlocks(M.f32, m, n, k, a_stride=stride, a_scale_stride=scale_stride, out_stride=out_stride)
    with Space((m - 1) * stride + k, 4 * ((m - 1) * scale_stride + 3), b.nbytes, 64, 4 * ((m - 1) * out_stride + n), max(16, op.workspace_bytes())) as s:
        for r in range(m):
            s.put(0, r * stride, a[r]), s.put(1, 4 * r * scale_stride, a_s[r].astype(np.float32))
        s.put(2, 0, b), s.put(3, 0, b_s.astype(np.float32))
        op.run_device([s.ptr(i) for i in range(6)])
        got = np.stack([s.get(4, 4 * r * out_stride, np.empty(n, np.float32)) for r in range(m)])
    a64, b64 = back(a, a_s, 1), back(b, b_s, 128)
    want = a64 @ b64.T
    assert (np.abs(got - want) <= product_bound(a64, b64, 3, HALF_STEP["f32"], want)).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_experts_far_apart(gpu, kind):
    """Three experts whose matrices lie more than 2^31 elements from each other."""
    layer = Layer(kind, 6, 256, 72, 3, 2, seed=4)
    size, apart = (2, 2200000016) if kind == "bf16" else (1, 2200000016)
    op = layer.op(gate_strides=(apart, 256), up_strides=(apart, 256), down_strides=(apart, 72))
    per = 72 * 256
    arrays = layer.arrays()
    small = [None if x is None else M.DeviceBuffer.from_numpy(x) for x in arrays]
    with Space(size * (2 * apart + 3 * per + 64), max(16, op.workspace_bytes())) as s:
        for j, name in enumerate(("gate", "up", "down")):   # one behind the other, expert after expert
            for e in range(3):
                s.put(0, size * (e * apart + j * per), layer.stored[name][e])
        pointers = [None if b is None else b.ptr for b in small] + [s.ptr(1)]
        for j in range(3):
            pointers[2 + j] = s.ptr(0) + size * j * per
        op.run_device(pointers)
        layer.check([small[i].to_numpy(arrays[i].dtype, arrays[i].shape) for i in (9, 10, 11)])
    for b in small:
        if b is not None:
            b.free()
