"""Products of tensors in e4m3 with a scale for each block, against the same in 64 bits."""
import numpy as np
import pytest

import morello_amd as M
from blocks_util import DTYPE, HALF_STEP, POISON, STORED, Device, as_f64, back, cast, product_bound, strided
from morello_amd import synth

pytestmark = pytest.mark.gpu


class Operands:
    def __init__(self, m, n, k, seed, narrow=False):
        """narrow: numbers of three binades, whose products' sums over a block need less than 13 bits below the largest: no instruction cuts them."""
        self.narrow, self.m, self.n, self.k, self.steps = narrow, m, n, k, -(-k // 128)
        a = synth.normal_f32(seed, 0, (m, k)).astype(np.float32)
        a[:, ::37] *= 20
        b = (synth.normal_f32(seed, 1, (n, k)) * k ** -0.5).astype(np.float32)
        (self.a, self.a_scales), (self.b, self.b_scales) = cast(a, 1), cast(b, 128)
        if narrow:
            self.a, self.b = ((0x40 + x % 24) | (x & 128) for x in (self.a, self.b))

    def want(self, out):
        a, b = back(self.a, self.a_scales, 1), back(self.b, self.b_scales, 128)
        c = a @ b.T
        return c, product_bound(a, b, self.steps, HALF_STEP[out], c, cut=out == "bf16" and not self.narrow)

    def run(self, out, a_stride=0, a_scale_stride=0, b_stride=0, b_scale_stride=0, out_stride=0, offset=0):
        """What lies between rows of a and b is NaN, between rows of out it is checked to be as it was; `offset`: of a and b, in bytes."""
        op = M.MatmulBlocks(DTYPE[out], self.m, self.n, self.k, a_stride, a_scale_stride, b_stride, b_scale_stride, out_stride)
        flat = {}
        for name, stride, fill, at in (("a", a_stride, 0x7f, offset), ("a_scales", a_scale_stride, np.nan, 0), ("b", b_stride, 0xff, offset), ("b_scales", b_scale_stride, np.nan, 0)):
            x = getattr(self, name)
            flat[name] = strided(x, stride or x.shape[1], fill, at)[0]
        five = np.full((self.m, self.n), {"bf16": 0x40a0, "f32": 5}[out], STORED[out])
        before, _ = strided(five, out_stride or self.n, POISON[out])
        with Device() as d:
            pointers = [d.put(flat["a"], offset), d.put(flat["a_scales"]), d.put(flat["b"], offset), d.put(flat["b_scales"]), d.put(before)]
            pointers.append(d.put(np.full(max(16, op.workspace_bytes()), 0xff, np.uint8)))
            op.run_device(pointers)
            after = d.get(4, before)
        view = lambda x: np.lib.stride_tricks.as_strided(x, five.shape, ((out_stride or self.n) * x.itemsize, x.itemsize))
        got = view(after).copy()
        view(after)[:] = five
        assert np.array_equal(after, before, equal_nan=out == "f32"), "written between the rows"
        return got

    def check(self, got, out):
        want, bound = self.want(out)
        off = np.abs(as_f64(out, got) - want)
        assert (off <= bound).all(), f"{(off / bound).max():.2f} of the bound, at {np.argwhere(~(off <= bound))[:4].tolist()}"


SIZES = [(20, 400, 1168), (38, 6200, 512), (50, 6160, 400), (77, 6200, 640), (90, 6150, 384), (90, 800, 1536), (72, 1000, 2048), (40, 100, 3000 + 8), (111, 250, 1024), (16, 33, 16),
         (1, 1, 1), (1, 16, 128), (1, 4096, 2048), (2, 17, 129), (7, 1000, 4104), (16, 512, 512), (17, 100, 1000), (32, 64, 257), (33, 130, 384), (48, 1040, 2176),
         (64, 64, 64), (65, 300, 130), (100, 2048, 1024), (128, 128, 128), (129, 257, 640), (200, 520, 15), (300, 200, 1111), (513, 384, 2048), (1000, 1030, 1200), (257, 2000, 33),
         (2049, 2050, 256), (600, 800, 1040),
         # tiles of 64 x 96, 96 x 64, 96 x 96 and 128 x 96, whole ones and ones that the sizes cut
         (1024, 1536, 400), (200, 6100, 272), (1536, 1024, 256), (1500, 1020, 1040), (1500, 1500, 528), (1001, 2050, 657), (1536, 1536, 128), (1537, 2000, 384), (2001, 1501, 1300),
         # workgroups that share K
         (97, 64, 3201), (129, 512, 3104), (130, 515, 4900), (200, 130, 8208), (600, 600, 3088), (97, 4096, 3090), (768, 520, 128), (1025, 513, 2000)]


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(gpu, m, n, k, out):
    x = Operands(m, n, k, m + n + k, narrow=m * n > 30000 or m % 2 == 1)
    x.check(x.run(out), out)


@pytest.mark.parametrize("m,n,k", [(33, 200, 512), (128, 128, 640), (300, 257, 400)])
def test_products_of_all_sizes_in_a_block(gpu, m, n, k):
    x = Operands(m, n, k, 9)
    x.check(x.run("bf16"), "bf16")


@pytest.mark.parametrize("m,n,k", [(5, 77, 300), (40, 150, 513), (150, 260, 400), (530, 700, 272)])
def test_strides_and_odd_addresses(gpu, m, n, k):
    x = Operands(m, n, k, 3, narrow=True)
    up = -(-k // 16) * 16 + 32
    for kw in (dict(a_stride=up, b_stride=up + 16, a_scale_stride=9, b_scale_stride=7, out_stride=n + 8), dict(a_stride=k + 3, b_stride=k + 1, offset=1, out_stride=n + 1),
               dict(a_stride=up, b_stride=k + 5, offset=8)):
        x.check(x.run("bf16", **kw), "bf16")
        x.check(x.run("f32", **kw), "f32")


@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_strides_where_workgroups_share_k(gpu, out):
    x = Operands(150, 130, 4000, 12, narrow=True)
    for kw in (dict(a_stride=4032, b_stride=4048, a_scale_stride=33, b_scale_stride=40, out_stride=138), dict(a_stride=4003, b_stride=4001, offset=1, out_stride=131), dict(a_stride=4032, b_stride=4005),
               dict(a_stride=4032, b_stride=4005, offset=8)):
        x.check(x.run(out, **kw), out)


@pytest.mark.parametrize("m,n,k", [(5, 70, 512), (60, 90, 512), (600, 530, 256)])
def test_rows_that_overlap(gpu, m, n, k):
    """Strides of inputs may be less than a row."""
    x = Operands(m, n, k, 10, narrow=True)
    flat_a, flat_b = x.a.reshape(-1)[:(m - 1) * 32 + k].copy(), x.b.reshape(-1)[:(n - 1) * 16 + k].copy()
    x.a = np.lib.stride_tricks.as_strided(flat_a, (m, k), (32, 1))
    x.b = np.lib.stride_tricks.as_strided(flat_b, (n, k), (16, 1))
    op = M.MatmulBlocks(M.bf16, m, n, k, a_stride=32, b_stride=16)
    out = np.zeros((m, n), np.uint16)
    with Device() as d:
        op.run_device([d.put(flat_a), d.put(x.a_scales), d.put(flat_b), d.put(x.b_scales), d.put(out), d.put(np.zeros(max(16, op.workspace_bytes()), np.uint8))])
        x.check(d.get(4, out), "bf16")


@pytest.mark.parametrize("m,n,k", [(3, 40, 300), (70, 200, 500), (260, 520, 640)])
def test_what_is_not_a_number_stays_in_its_row_and_column(gpu, m, n, k):
    x = Operands(m, n, k, 4)
    x.a[m // 2, k - 1], x.b[n // 3, 0] = 0x7f, 0xff
    got = as_f64("f32", x.run("f32"))
    nan = np.zeros((m, n), bool)
    nan[m // 2], nan[:, n // 3] = True, True
    want, bound = x.want("f32")
    assert np.isnan(got[nan]).all() and (np.abs(got - want) <= bound)[~nan].all()


@pytest.mark.parametrize("m,n,k", [(4, 64, 1024), (90, 128, 1024), (300, 300, 1024)])
def test_scales_far_apart(gpu, m, n, k):
    """Blocks of K whose scales differ by 2^60 and more, and one of which is zero: each block's sums are multiplied by its own."""
    x = Operands(m, n, k, 5)
    for q in range(x.steps):
        x.a_scales[:, q] *= np.float32(2.0 ** (-60 + 15 * q))
    x.b_scales[:, 3] = 0
    x.check(x.run("f32"), "f32")


def test_repeats_bit_for_bit(gpu):
    for m, n, k in ((8, 4096, 4096), (70, 1500, 3000), (400, 1100, 1024), (130, 200, 5000)):
        x = Operands(m, n, k, 6)
        first = x.run("f32")
        assert np.array_equal(first, x.run("f32"))


@pytest.mark.parametrize("m,n,k", [(1, 100, 2064), (2, 3000, 1001), (3, 3000, 1001), (16, 130, 1000), (17, 77, 384), (32, 200, 1040), (33, 130, 272), (150, 300, 400)])
def test_whole_chunks_at_odd_addresses(gpu, m, n, k):
    """Strides that say whole chunks of addresses that are not: the sizes alone decide on the workspace."""
    x = Operands(m, n, k, 11, narrow=True)
    up = -(-k // 16) * 16
    for offset in (1, 8):
        for kw in (dict(a_stride=up, b_stride=up), dict(a_stride=up, b_stride=up + 3), dict(a_stride=k + 1, b_stride=up)):
            for out in ("bf16", "f32"):
                x.check(x.run(out, offset=offset, **kw), out)


# On tiles of 256 x 256 (130 to 169 of them): blocks of K that the ring's two and the scales' eight go around once and more, whole last ones and cut ones; scales of a in fours (blocks a multiple of four) and one by one
WIDE = [(3100, 3100, 1200), (3100, 3101, 1424), (3099, 3100, 2304), (3100, 3100, 2560), (3100, 3100, 1300), (3090, 3100, 128), (3100, 3090, 272), (3100, 3100, 4096),
        (130, 33104, 272), (2049, 4096, 400), (2944, 2888, 1424)]
# On tiles of 128 x 64, and past a round of 128 x 128, of many blocks
MORE_TILES = [(1280, 1216, 400), (1279, 1217, 1552), (1280, 1216, 1024), (2049, 2050, 1168), (2049, 2050, 1024), (2170, 2060, 1300)]


@pytest.mark.parametrize("m,n,k", WIDE)
def test_product_on_wide_tiles(gpu, m, n, k):
    x = Operands(m, n, k, m + n + k, narrow=True)
    first = x.run("bf16")
    x.check(first, "bf16")
    assert np.array_equal(first, x.run("bf16"))


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", MORE_TILES)
def test_product_on_more_tiles(gpu, m, n, k, out):
    x = Operands(m, n, k, m + n + k, narrow=True)
    x.check(x.run(out), out)


@pytest.mark.parametrize("k,a_scale_stride", [(1424, 13), (1424, 16), (2560, 21), (1200, 12)])
def test_strides_on_wide_tiles(gpu, k, a_scale_stride):
    x = Operands(3100, 3100, k, 13, narrow=True)
    x.check(x.run("bf16", a_stride=k + 32, b_stride=k + 16, a_scale_stride=a_scale_stride, b_scale_stride=a_scale_stride + 3, out_stride=3109), "bf16")


@pytest.mark.parametrize("k", [1424, 1200])
def test_scales_far_apart_on_wide_tiles(gpu, k):
    """Every block of K has a scale of its own, by 2^10 apart: none is multiplied by another's."""
    x = Operands(3100, 3100, k, 14, narrow=True)
    for q in range(x.steps):
        x.a_scales[:, q] *= np.float32(2.0 ** (10 * (q % 5) - 20))
        x.b_scales[:, q] *= np.float32(2.0 ** (7 * (q % 3) - 7))
    x.check(x.run("bf16"), "bf16")


@pytest.mark.parametrize("k", [1424, 1200])
def test_what_is_not_a_number_on_wide_tiles(gpu, k):
    m = n = 3100
    x = Operands(m, n, k, 15, narrow=True)
    x.a[m - 1, k - 1], x.a[300, 0], x.b[n // 3, k - 17] = 0x7f, 0xff, 0xff
    got = as_f64("bf16", x.run("bf16"))
    nan = np.zeros((m, n), bool)
    nan[[m - 1, 300]], nan[:, n // 3] = True, True
    assert np.array_equal(np.isnan(got), nan)
