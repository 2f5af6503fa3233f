"""Tensors in e4m3 with a scale for each block, and layers of experts: the operators' definitions in numpy (no code of the library)."""
import numpy as np

import morello_amd as M
from morello_amd import synth
from paged_util import DTYPE, HALF_STEP, POISON, STORED, as_f64, values  # noqa: F401

U = 2.0 ** -24   # half a step of 32 bits, relative


def _table():
    """What each byte stands for: sign, four bits of exponent (bias 7), three of mantissa; all ones is NaN."""
    code = np.arange(256)
    e, m = code >> 3 & 15, code & 7
    size = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    size = np.where(code & 127 == 127, np.nan, size)
    return np.where(code & 128, -size, size)


E4M3 = _table()
_POSITIVE = E4M3[:127]


def nearest_e4m3(x):
    """Bytes of the nearest numbers, of two equally near the one whose byte is even."""
    x = np.asarray(x, np.float64)
    size = np.minimum(np.abs(x), 448.0)
    hi = np.clip(np.searchsorted(_POSITIVE, np.nan_to_num(size)), 1, 126)
    lo = hi - 1
    down, up = size - _POSITIVE[lo], _POSITIVE[hi] - size
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.isnan(x), 127, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def over_blocks(scales, rows, cols, high):
    return np.repeat(np.repeat(scales, high, -2)[..., :rows, :], 128, -1)[..., :cols]


def cast(x, high):
    """x in f32 -> (bytes, scales): the definition, step by step in 32 bits."""
    x = np.asarray(x, np.float32)
    rows, cols = x.shape
    padded = np.zeros((-(-rows // high) * high, -(-cols // 128) * 128), np.float32)
    padded[:rows, :cols] = np.where(np.isnan(x), 0, np.abs(x))
    a = padded.reshape(-1, high, padded.shape[1] // 128, 128).max((1, 3))
    a = np.maximum(a, np.float32(2.0 ** -110))
    with np.errstate(invalid="ignore"):
        product = x * over_blocks(np.float32(448) / a, rows, cols, high)
    return nearest_e4m3(product), a / np.float32(448)


def back(stored, scales, high):
    """What bytes and scales stand for, in 64 bits."""
    return E4M3[stored] * over_blocks(scales.astype(np.float64), *stored.shape[-2:], high)


def strided(array, stride, fill, offset=0):
    """A buffer that holds the rows `stride` elements apart, `offset` elements in, and the buffer's view of them."""
    rows, cols = array.shape
    flat = np.full(offset + (rows - 1) * stride + max(cols, stride), fill, array.dtype)
    view = np.lib.stride_tricks.as_strided(flat[offset:], array.shape, (stride * array.itemsize, array.itemsize))
    view[:] = array
    return flat, view


class Device:
    """Arrays in device memory for the length of a test."""

    def __init__(self):
        self.bufs = []

    def put(self, array, offset=0):
        """-> the address of the array's element `offset`."""
        b = M.DeviceBuffer.from_numpy(np.ascontiguousarray(array))
        self.bufs.append(b)
        return b.ptr + offset * array.itemsize

    def get(self, i, like):
        return self.bufs[i].to_numpy(like.dtype, like.shape)

    def __enter__(self):
        return self

    def __exit__(self, *_):
        for b in self.bufs:
            b.free()


def product_bound(a64, b64, steps, half, want, cut=False):
    """How far the product may be off: a matrix instruction's sums over 128 products (exact, or cut to 32 bits one by one: 2 u each), the product of the scales and of it
    with the sums, a rounding for each block's addition, and as many again where waves or pieces share the blocks; then the result's.  `cut`: every
    product may lose 2^-13 of its block's largest."""
    bound = (2 * 128 + 2 * steps + 8) * U * (np.abs(a64) @ np.abs(b64).T)
    for q in range(0, a64.shape[1] if cut else 0, 128):
        a, b = np.abs(a64[:, q:q + 128]), np.abs(b64[:, q:q + 128])
        for i in range(len(a)):
            p = a[i] * b
            bound[i] += np.minimum(p, p.max(1, keepdims=True) * 2.0 ** -13).sum(1)
    return bound * (1 + half) + half * np.abs(want)


class Layer:
    """A layer of experts with its inputs, and what comes out of it."""

    def __init__(self, kind, tokens, hidden, inter, experts, top_k, seed, renormalise=False):
        self.kind, self.tokens, self.hidden, self.inter, self.experts, self.top_k, self.renormalise = kind, tokens, hidden, inter, experts, top_k, renormalise
        self.x, self.x64 = values("bf16", seed, 0, (tokens, hidden))
        self.router, self.router64 = values("bf16", seed, 1, (experts, hidden), 1.5 * hidden ** -0.5)
        self.stored, self.scales, self.w64 = {}, {}, {}
        for i, (name, rows, cols) in enumerate((("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter))):
            if kind == "bf16":
                self.stored[name], self.w64[name] = values("bf16", seed, 2 + i, (experts, rows, cols), cols ** -0.5)
                continue
            w = (synth.normal_f32(seed, 2 + i, (experts, rows, cols)) * cols ** -0.5).astype(np.float32)
            both = [cast(w[e], 128) for e in range(experts)]
            self.stored[name], self.scales[name] = np.stack([b for b, _ in both]), np.stack([s for _, s in both])
            self.w64[name] = np.stack([back(b, s, 128) for b, s in both])

    def op(self, **given):
        kwargs = dict(tokens=self.tokens, hidden=self.hidden, inter=self.inter, experts=self.experts, top_k=self.top_k, renormalise=self.renormalise)
        kwargs.update(given)
        return M.Experts(M.bf16 if self.kind == "bf16" else M.f8e4m3, **kwargs)

    def choice(self):
        """(experts, shares): by logits in 64 bits, of equal ones the lowest."""
        logits = self.x64 @ self.router64.T
        order = np.argsort(-logits, 1, kind="stable")[:, :self.top_k]
        p = np.exp(logits - logits.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        shares = np.take_along_axis(p, order, 1)
        return order, shares / shares.sum(1, keepdims=True) if self.renormalise else shares

    def want(self, rows=None, h_step=2.0 ** -8):
        """(out, bound, chosen, shares).  A sum of n products is off by at most 2 n u times the sum of their sizes (in any order, with a share of it
        for blocks and pieces); silu's derivative is at most 1.1 and its own steps good to 8 u; h is rounded by h_step: bf16's, or 2^-16 for two such numbers; shares are good to 1e-6."""
        rows = self.tokens if rows is None else rows
        chosen, shares = self.choice()
        out, bound = np.zeros((rows, self.hidden)), np.zeros((rows, self.hidden))
        for t in range(rows):
            for e, share in zip(chosen[t], shares[t]):
                gate, up, down = (self.w64[n][e] for n in ("gate", "up", "down"))
                x = self.x64[t]
                g, u = gate @ x, up @ x
                n = 2 * (self.hidden + 64) * U
                eg, eu = n * (np.abs(gate) @ np.abs(x)), n * (np.abs(up) @ np.abs(x))
                silu = g / (1 + np.exp(-g))
                h = silu * u
                eh = 1.1 * eg * (np.abs(u) + eu) + np.abs(silu) * eu + (8 * U + h_step) * (np.abs(h) + 1.1 * eg * np.abs(u) + np.abs(silu) * eu)
                out[t] += share * (down @ h)
                bound[t] += share * (np.abs(down) @ eh + (2 * (self.inter + 64) * U + 2e-6) * (np.abs(down) @ (np.abs(h) + eh)))
        half = HALF_STEP["bf16"]
        return out, bound * (1 + half) + half * np.abs(out), chosen[:rows], shares[:rows]

    def arrays(self):
        """In the order of the call's parameters, None where there is none; out, chosen and shares of a poison each."""
        scales = [self.scales.get(n) for n in ("gate", "up", "down")]
        return [self.x, self.router] + [self.stored[n] for n in ("gate", "up", "down")] + scales + [
            None, np.full((self.tokens, self.hidden), POISON["bf16"], np.uint16), np.full((self.tokens, self.top_k), -7, np.int32),
            np.full((self.tokens, self.top_k), np.nan, np.float32)]

    def run(self, op=None, rows=None):
        """-> out (stored), chosen, shares."""
        op = op or self.op()
        arrays = self.arrays()
        if rows is not None:
            arrays[8] = np.array([rows], np.int32)
        arrays.append(np.full(max(16, op.workspace_bytes()), 0xff, np.uint8))   # (NaN, -1: what it holds does not matter)
        with Device() as d:
            at, pointers = {}, []
            for i, a in enumerate(arrays):
                if a is not None:
                    at[i] = len(d.bufs)
                pointers.append(None if a is None else d.put(a))
            op.run_device(pointers)
            return [d.get(at[i], arrays[i]) for i in (9, 10, 11)]

    def check(self, got, rows=None):
        out, chosen, shares = got
        n = self.tokens if rows is None else max(0, min(rows, self.tokens))
        want, bound, which, parts = self.want(n)
        assert np.array_equal(chosen[:n], which)
        assert np.abs(shares[:n] / parts - 1).max(initial=0) <= 1e-6
        off = np.abs(as_f64("bf16", out[:n]) - want)
        assert (off <= bound).all(), f"{(off / bound).max():.2f} of the bound, at {np.argwhere(~(off <= bound))[:4].tolist()}"
        assert (out[n:] == POISON["bf16"]).all() and (chosen[n:] == -7).all() and np.isnan(shares[n:]).all(), "rows behind the last were written"
