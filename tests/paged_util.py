"""Batches over a cache of keys and values in pages, and the operators' definitions in 64 bits (numpy, no code of the library)."""
import numpy as np

import morello_amd as M
from morello_amd import synth

HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}   # of a rounding, relative
DTYPE = {"bf16": M.bf16, "f32": M.f32}
POISON = {"bf16": np.uint16(0x7fc0), "f32": np.float32(np.nan)}
STORED = {"bf16": np.uint16, "f32": np.float32}


def values(dtype, seed, index, shape, std=1.0):
    """Stored values of a tensor and the same in 64 bits."""
    if dtype == "bf16":
        bits = synth.normal_bf16(seed, index, shape, std)
        return bits, synth.bf16_bits_to_f32(bits).astype(np.float64)
    x = (synth.normal_f32(seed, index, shape) * std).astype(np.float32)
    return x, x.astype(np.float64)


def as_f64(dtype, stored):
    return (synth.bf16_bits_to_f32(stored) if dtype == "bf16" else stored).astype(np.float64)


class Batch:
    """`lengths`: (tokens in the cache, new ones) of each request.  Every slot that no request's key is in holds NaN."""

    def __init__(self, dtype, lengths, q_heads, kv_heads, dim, page, seed, heads_first=False, spare_rows=3, q_std=2.0, first=0):
        self.dtype, self.lengths, self.q_heads, self.kv_heads, self.dim, self.page = dtype, lengths, q_heads, kv_heads, dim, page
        rng = np.random.default_rng(seed)
        need = [-(-(c + n) // page) for c, n in lengths]
        self.pages, self.width = sum(need) + 3, max(max(need), 1) + 1
        self.requests = len(lengths)
        ids = rng.permutation(self.pages)
        self.table = np.full((self.requests, self.width), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = ids[at:at + n]
            at += n
        self.starts = (first + np.concatenate([[0], np.cumsum([n for _, n in lengths])])).astype(np.int32)
        self.totals = np.array([c + n for c, n in lengths], np.int32)
        self.tokens = int(self.starts[-1]) + spare_rows
        self.heads_first = heads_first
        shape = (self.pages, kv_heads, page, dim) if heads_first else (self.pages, page, kv_heads, dim)
        self.strides = (kv_heads * page * dim, dim, page * dim) if heads_first else (page * kv_heads * dim, kv_heads * dim, dim)
        self.q, self.q64 = values(dtype, seed, 0, (self.tokens, q_heads, dim), q_std)
        self.q[:first], self.q[self.starts[-1]:] = POISON[dtype], POISON[dtype]
        self.keys, self.values = (values(dtype, seed, i, shape)[0] for i in (1, 2))
        used = np.zeros((self.pages, page), bool)
        for r, (c, n) in enumerate(lengths):
            for j in range(need[r]):
                used[self.table[r, j], :min(page, c + n - j * page)] = True
        for cache in (self.keys, self.values):
            (cache.transpose(0, 2, 1, 3) if heads_first else cache)[~used] = POISON[dtype]

    def op(self, **given):
        kwargs = dict(tokens=self.tokens, requests=self.requests, q_heads=self.q_heads, kv_heads=self.kv_heads, head_dim=self.dim,
                      page_size=self.page, pages=self.pages, table_width=self.width, max_new=max(1, max(n for _, n in self.lengths)),
                      key_strides=self.strides, value_strides=self.strides)
        kwargs.update(given)
        return M.PagedAttention(DTYPE[self.dtype], **kwargs)

    def rows(self, cache):
        c = as_f64(self.dtype, cache)
        return c.transpose(0, 2, 1, 3) if self.heads_first else c   # [page][slot][head][dim]

    def want(self, window=0, scale=None):
        """(out, bound): the formula, and how far each element may be off.  With p_j the probabilities, A = sum_j p_j |v_j| and
        u the half step of 32 bits:
          - a score is a sum of dim products of numbers that are rounded once more by the scale: off by at most (dim + 4) u scale |q|.|k|;
          - its exponential takes s - m in the base of 2, which rounds by at most 4 u (|s| + |m|), and is good to 4 u itself;
          - so each p_j is off by at most d relative, d the sum of these, and sum and quotient by twice that; the sums over n keys by n u;
          - bf16: p_j is rounded for the second product (2^-8), in numerator and denominator alike;
          - the result is rounded once."""
        scale = self.dim ** -0.5 if scale is None else scale
        u, half = 2.0 ** -24, HALF_STEP[self.dtype]
        out = np.zeros((self.tokens, self.q_heads, self.dim))
        bound = np.zeros_like(out)
        keys, vals = self.rows(self.keys), self.rows(self.values)
        for r in range(self.requests):
            start, end, length = int(self.starts[r]), int(self.starts[r + 1]), int(self.totals[r])
            j = np.arange(min(max(length, 0), self.width * self.page))
            numbers = self.table[r, j // self.page]
            there = (numbers >= 0) & (numbers < self.pages)
            j, numbers = j[there], numbers[there]
            k, v = keys[numbers, j % self.page], vals[numbers, j % self.page]
            for t in range(start, end):
                p = length - (end - t)
                seen = (j <= p) & ((j > p - window) if window else True)
                if not seen.any():
                    continue
                ks, vs = k[seen], v[seen]
                for h in range(self.q_heads):
                    g = h // (self.q_heads // self.kv_heads)
                    q = self.q64[t, h]
                    s = scale * (ks[:, g] @ q)
                    left = s != -np.inf   # (a score of -infinity weighs nothing)
                    if not left.any():
                        continue
                    s, kg, vg = s[left], ks[left, g], vs[left, g]
                    size = scale * (np.abs(kg) @ np.abs(q))
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[t, h] = w @ vg
                    a = w @ np.abs(vg)
                    d = (self.dim + 4) * u * abs(size).max() + 4 * u * 2 * np.abs(s).max() + 4 * u + (2.0 ** -8 if self.dtype == "bf16" else 0.0)
                    bound[t, h] = half * np.abs(out[t, h]) + (1 + half) * (2 * d + 2 * len(s) * u) * a
        return out, bound

    def run(self, op, stream=None, out=None, table=None):
        """-> what the call left in `out` (stored values), 5 everywhere before."""
        five = {"bf16": np.uint16(0x40a0), "f32": np.float32(5)}[self.dtype]
        host_out = np.full((self.tokens, self.q_heads, self.dim), five, STORED[self.dtype]) if out is None else out
        bufs = [M.DeviceBuffer.from_numpy(a) for a in (self.q, self.keys, self.values, self.table if table is None else table, self.starts, self.totals, host_out)]
        bytes_ = op.workspace_bytes()
        bufs.append(M.DeviceBuffer.from_numpy(np.full(max(bytes_, 16), 0xff, np.uint8)))   # (NaN, -1: what it holds does not matter)
        op.run_device([b.ptr for b in bufs])
        got = bufs[6].to_numpy(host_out.dtype, host_out.shape)
        for b in bufs:
            b.free()
        return got

    def check(self, got, window=0, scale=None):
        want, bound = self.want(window, scale)
        g = as_f64(self.dtype, got)
        first, end = int(self.starts[0]), int(self.starts[-1])
        assert (g[:first] == 5).all() and (g[end:] == 5).all(), "rows of no request were written"
        off = np.abs(g[first:end] - want[first:end])
        assert np.isfinite(g[first:end]).all(), f"not finite: {np.argwhere(~np.isfinite(g[first:end]))[:4].tolist()}"
        worst = (off / np.maximum(bound[first:end], 1e-300)).max(initial=0.0) if end > first else 0.0
        assert (off <= bound[first:end]).all(), f"{worst:.2f} of the bound, at {np.argwhere(off > bound[first:end])[:4].tolist()}"
        return worst
