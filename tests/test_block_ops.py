"""Descriptors of the operators on blocks of e4m3 and of experts: what is refused, and which kernels a call would launch.  No GPU needed."""
import ctypes as C

import numpy as np
import pytest

import morello_amd as M
from blocks_util import E4M3, back, cast, nearest_e4m3
from morello_amd import _binding as B

OK, UNSUPPORTED, BAD_SPEC, NULL, TOO_LARGE = 0, 1, 3, 6, 7


def cast_op(dtype=M.bf16, **given):
    return M.CastBlocks(dtype, **{**dict(rows=33, cols=300), **given})


def product(dtype=M.bf16, **given):
    return M.MatmulBlocks(dtype, **{**dict(m=33, n=200, k=300), **given})


def experts(dtype=M.f8e4m3, **given):
    return M.Experts(dtype, **{**dict(tokens=4, hidden=256, inter=128, experts=16, top_k=2), **given})


def test_struct_sizes_match_the_header():
    assert C.sizeof(B.CastBlocksC) == 6 * 4 + 3 * 8
    assert C.sizeof(B.MatmulBlocksC) == 4 * 4 + 5 * 8
    assert C.sizeof(B.ExpertsC) == 8 * 4 + 3 * 8 + 12 * 8


def test_the_type_of_eight_bits():
    assert M.f8e4m3.size == 1 and str(M.f8e4m3) == "f8e4m3"
    assert M.Matmul([1, 4, 4, 4], [M.f8e4m3] * 3).check() == BAD_SPEC


def test_the_type_of_eight_bits_is_of_no_spec():
    """What a search asks about Specs knows as little of it as of numbers that are no type."""
    for dtype in (M.f8e4m3, 9, -1):
        assert M.Target.all_layouts_for_shape([64, 64], dtype) == []
    lib = B.load()
    spec = M.Matmul([1, 4, 4, 4], [M.u8, M.f8e4m3, M.i32])
    assert [lib.mrl_spec_parameter_bytes(C.byref(spec._c), i) for i in range(3)] == [16, 0, 64]


@pytest.mark.parametrize("given,status", [
    (dict(), OK), (dict(dtype=M.f32), OK), (dict(dtype=M.i8), UNSUPPORTED), (dict(dtype=M.f8e4m3), BAD_SPEC), (dict(dtype=99), BAD_SPEC), (dict(rows=0), BAD_SPEC), (dict(cols=0), BAD_SPEC),
    (dict(block_rows=128), OK), (dict(block_rows=0), BAD_SPEC), (dict(block_rows=64), BAD_SPEC), (dict(rows=1 << 27, cols=128), OK), (dict(rows=1 << 27, cols=129), TOO_LARGE),
    (dict(rows=1, cols=0xffffffff), TOO_LARGE), (dict(rows=1, cols=(1 << 30) - 1, gated=True), OK), (dict(x_stride=7), OK), (dict(x_stride=-1), BAD_SPEC),
    (dict(out_stride=299), BAD_SPEC), (dict(out_stride=300), OK), (dict(scale_stride=2), BAD_SPEC), (dict(scale_stride=3), OK), (dict(rows=1, out_stride=1), OK),
    (dict(x_stride=(1 << 40) + 1), BAD_SPEC), (dict(rows=1 << 24, x_stride=1 << 40), TOO_LARGE),
])
def test_cast_blocks_check(given, status):
    assert cast_op(**given).check() == status


@pytest.mark.parametrize("given,status", [
    (dict(), OK), (dict(dtype=M.f32), OK), (dict(dtype=M.u16), UNSUPPORTED), (dict(dtype=-1), BAD_SPEC), (dict(dtype=M.f8e4m3), BAD_SPEC), (dict(m=0), BAD_SPEC), (dict(n=0), BAD_SPEC),
    (dict(k=0), BAD_SPEC), (dict(m=1 << 23, n=1 << 17), OK), (dict(m=1 << 23, n=(1 << 17) + 1), TOO_LARGE), (dict(m=(1 << 23) + 1), TOO_LARGE), (dict(n=(1 << 23) + 1), TOO_LARGE),
    (dict(k=(1 << 23) + 1), TOO_LARGE), (dict(out_stride=199), BAD_SPEC), (dict(a_stride=1, a_scale_stride=1, b_stride=1, b_scale_stride=1), OK), (dict(b_stride=-5), BAD_SPEC),
])
def test_matmul_blocks_check(given, status):
    op = product(**given)
    assert op.check() == status
    if status != OK:
        assert op.workspace_bytes() == 0
        with pytest.raises(M.MorelloError) as err:
            op.plan()
        assert err.value.status == status


@pytest.mark.parametrize("given,status", [
    (dict(), OK), (dict(dtype=M.bf16), OK), (dict(dtype=M.f32), UNSUPPORTED), (dict(dtype=9), BAD_SPEC), (dict(tokens=0), BAD_SPEC), (dict(tokens=256), OK), (dict(tokens=257), TOO_LARGE),
    (dict(hidden=0), BAD_SPEC), (dict(inter=0), BAD_SPEC), (dict(experts=0), BAD_SPEC), (dict(experts=512), OK), (dict(experts=513), TOO_LARGE), (dict(top_k=0), BAD_SPEC),
    (dict(top_k=17), BAD_SPEC), (dict(experts=64, top_k=32), OK), (dict(experts=64, top_k=33), TOO_LARGE), (dict(hidden=1 << 17), OK), (dict(hidden=(1 << 17) + 1), TOO_LARGE),
    (dict(inter=(1 << 17) + 1), TOO_LARGE), (dict(out_stride=255), BAD_SPEC), (dict(x_stride=0, out_stride=256), OK), (dict(gate_strides=(0, 256)), OK), (dict(gate_strides=(-1, 256)), BAD_SPEC),
    (dict(down_scale_strides=(1 << 41, 1)), BAD_SPEC), (dict(dtype=M.bf16, down_scale_strides=(1 << 41, 1)), OK),
])
def test_experts_check(given, status):
    op = experts(**given)
    assert op.check() == status
    assert (op.workspace_bytes() > 0) == (status == OK)


def test_null_descriptors_and_lists():
    lib = B.load()
    for name in ("cast_blocks", "matmul_blocks", "experts"):
        assert getattr(lib, f"mrl_{name}_check")(None) == NULL
        assert getattr(lib, f"mrl_run_{name}")(None, None, None) == NULL
        assert getattr(lib, f"mrl_{name}_plan")(None, None, None, 0) == NULL
    for op in (cast_op(), product(), experts()):
        assert op._run(C.byref(op._c), None, None) == NULL
        with pytest.raises(ValueError):
            op.run_async([1, 2])
    with pytest.raises(ValueError):
        experts(gate_strides=(1, 2, 3))


def test_plans():
    families = set(M.Target.kernels())
    for op in (cast_op(), cast_op(M.f32, gated=True, block_rows=128), product(), product(M.f32, m=4), product(m=4096, n=4096, k=4096), experts(), experts(M.bf16, tokens=256)):
        plan = op.plan()
        assert plan.steps and set(plan.kernels) <= families and plan.cost_ns >= 2000 * len(plan.steps), plan
    assert product().plan().scratch_bytes == product().workspace_bytes()
    assert experts().plan().scratch_bytes == experts().workspace_bytes()


ODD = dict(a_stride=4097)


@pytest.mark.parametrize("m,n,k,out,strides,kernel,copied", [
    (1, 4096, 4096, M.bf16, {}, "k_product_few", 0), (96, 4096, 4096, M.f32, {}, "k_product_few", 0), (97, 8192, 4096, M.bf16, {}, "k_product_tile", 0),
    (4096, 4096, 4096, M.bf16, {}, "k_product_wide", 0), (4096, 4096, 4096, M.f32, {}, "k_product_tile", 0), (2048, 4096, 4096, M.bf16, {}, "k_product_tile", 0),
    (2048, 6144, 4096, M.bf16, {}, "k_product_wide", 0), (16, 100, 4095, M.bf16, {}, "k_product_few_any", 0), (17, 100, 4095, M.bf16, {}, "k_product_few", 117 * 4096),
    (2, 4000, 4095, M.f32, {}, "k_product_few_any", 0), (3, 4000, 4095, M.f32, {}, "k_product_few", 4003 * 4096),
    (40, 100, 4096, M.bf16, ODD, "k_product_few", 40 * 4096), (40, 100, 4096, M.bf16, dict(b_stride=4100), "k_product_few", 100 * 4096),
    (100, 1 << 23, 2049, M.bf16, {}, "k_product_tile_any", 0), (300, 100, 256, M.f32, dict(a_scale_stride=1 << 21), "k_product_tile_any", 0),
])
def test_which_kernel_a_product_takes(m, n, k, out, strides, kernel, copied):
    op = M.MatmulBlocks(out, m, n, k, **strides)
    assert op.workspace_bytes() == copied
    steps = op.plan().steps
    assert [s.family for s in steps][-1] == kernel and len(steps) == 1 + (copied > 0)


@pytest.mark.parametrize("m,n,k,kernel", [
    (2048, 4096, 4096, "k_product_tile"), (2049, 4096, 4096, "k_product_wide"), (2304, 4096, 1024, "k_product_wide"), (3000, 3000, 2000, "k_product_wide"), (2816, 2816, 2048, "k_product_tile"),
    (2944, 2944, 2048, "k_product_wide"), (4608, 4096, 512, "k_product_tile"), (5120, 4096, 4096, "k_product_wide"), (2000, 16384, 512, "k_product_wide"), (130, 40000, 256, "k_product_wide"),
    (2900, 2950, 1040, "k_product_tile"), (3100, 3100, 1040, "k_product_wide")])
def test_where_products_take_wide_tiles(m, n, k, kernel):
    """In one round of them where the smaller tiles make more than one; past a round, and of results whose rows are off 16 bytes, where the last is full enough."""
    assert [s.family for s in M.MatmulBlocks(M.bf16, m, n, k).plan().steps] == [kernel]
    assert [s.family for s in M.MatmulBlocks(M.f32, m, n, k).plan().steps] == ["k_product_tile"]


@pytest.mark.parametrize("m,n,k,strides,shares,copied", [
    (97, 4096, 4096, {}, 2, 0), (97, 4097, 4096, {}, 1, 0), (128, 512, 1535, {}, 1, 640 * 1536), (128, 512, 3200, {}, 2, 0), (129, 510, 4992, {}, 3, 0), (200, 130, 8192, dict(a_stride=8193), 5, 200 * 8192), (96, 512, 8192, {}, 1, 0)])
def test_few_tiles_share_k(m, n, k, strides, shares, copied):
    op = M.MatmulBlocks(M.f32, m, n, k, **strides)
    assert op.workspace_bytes() == copied + (shares * m * (-(-n // 4) * 4) * 4 if shares > 1 else 0)
    assert [s.family for s in op.plan().steps][copied > 0:] == (["k_product_tile", "k_product_join"] if shares > 1 else ["k_product_tile"] if m > 96 else ["k_product_few"])


@pytest.mark.parametrize("tokens,hidden,experts_,top_k,launches", [
    (1, 2048, 181, 8, 3), (1, 2048, 182, 8, 4), (8, 2048, 32, 8, 3), (8, 2048, 33, 8, 4), (32, 2048, 8, 1, 3), (33, 2048, 7, 1, 4), (32, 2048, 8, 2, 4), (256, 2048, 512, 32, 4)])
def test_which_kernels_a_layer_of_experts_takes(tokens, hidden, experts_, top_k, launches):
    for dtype in (M.bf16, M.f8e4m3):
        families = [s.family for s in M.Experts(dtype, tokens, hidden, 768, experts_, top_k).plan().steps]
        assert families == ["k_experts_logits"] + ["k_experts_choose"] * (launches == 4) + ["k_experts_up", "k_experts_down"]


@pytest.mark.parametrize("hidden,inter,joined", [(1024, 2048, True), (1024, 512, False), (2048, 1 << 15, False), (1032, 1 << 15, False), (384, 9600, True)])
def test_few_rows_of_down_are_shared(hidden, inter, joined):
    op = M.Experts(M.bf16, 1, hidden, inter, 64, 8)
    assert ([s.family for s in op.plan().steps][-1] == "k_experts_join") == joined
    assert (op.workspace_bytes() >= 2 * hidden * 4) or not joined


def test_values_are_compared_of_every_form_of_the_kernels():
    """The sizes whose results are compared with the oracle's reach every kernel that the library chooses between, with all its template arguments."""
    import test_gpu_experts as E
    import test_gpu_matmul_blocks as P

    ops = [M.MatmulBlocks(out, *s) for out in (M.bf16, M.f32) for s in P.SIZES + P.MORE_TILES] + [M.MatmulBlocks(M.bf16, *s) for s in P.WIDE]
    ops += [M.Experts(kind, *s) for kind in (M.bf16, M.f8e4m3) for s in E.SIZES + E.MORE]
    reached = {s.kernel for op in ops for s in op.plan().steps}
    tiles = [(128, 128, 1, 2), (128, 128, 2, 2), (128, 96, 2, 2), (128, 64, 2, 3), (96, 96, 2, 3), (96, 64, 2, 3), (64, 96, 2, 3), (64, 64, 3, 3)]
    few = [(1, 1, 8, 4), (2, 1, 8, 3), (3, 1, 8, 2), (3, 2, 4, 3), (4, 1, 4, 3), (4, 2, 4, 3), (5, 1, 6, 2), (5, 2, 4, 2), (6, 1, 4, 2), (6, 2, 4, 2)]
    want = {f"k_product_wide [CHUNKS = {c}]" for c in ("false", "true")}
    for out in ("float", "unsigned short"):
        want |= {"k_product_tile [BM = %d, BN = %d, GROUPS = %d, DEPTH = %d, OUT = %s, SHARED = false]" % (*t, out) for t in tiles}
        want |= {f"k_product_tile [BM = 64, BN = 64, GROUPS = 3, DEPTH = 3, OUT = {out}, SHARED = true]", f"k_product_join [OUT = {out}]", f"k_product_few_any [OUT = {out}]"}
        want |= {"k_product_few [MT = %d, NT = %d, WAVES = %d, DEPTH = %d, OUT = %s]" % (*f, out) for f in few}
    for f8 in ("false", "true"):
        for tail in range(3):
            want |= {f"k_experts_up [F8 = {f8}, ROOM = 16, FUSED = false, TAIL = {tail}, UP_WAVES = 4]"}
            want |= {f"k_experts_up [F8 = {f8}, ROOM = 8, FUSED = {fused}, TAIL = {tail}, UP_WAVES = {waves}]" for fused in ("false", "true") for waves in (4, 8) if (waves, tail) != (8, 2)}
            want |= {f"k_experts_down [F8 = {f8}, MOST = 16, TAIL = {tail}, HOW = 0]"}
            want |= {f"k_experts_down [F8 = {f8}, MOST = 4, TAIL = {tail}, HOW = {how}]" for how in range(3) if (how, tail) != (2, 2)}
    assert want <= reached, sorted(want - reached)
    assert {k for k in reached - want if "[" in k and not k.startswith(("k_experts_logits", "k_pad_rows"))} == set()


def test_the_oracle_of_the_casts():
    """Every byte is its own nearest; between two numbers the nearer, halfway the even byte; a block reads back within half a step."""
    codes = np.array([c for c in range(256) if c & 127 != 127])
    assert np.array_equal(nearest_e4m3(E4M3[codes]), codes)
    assert E4M3[0x7e] == 448 and E4M3[0x08] == 2.0 ** -6 and E4M3[0x01] == 2.0 ** -9 and np.isnan(E4M3[0x7f])
    assert nearest_e4m3([17, 19, 2.0 ** -10, 1.5 * 2.0 ** -9, 447, 460, -0.0]).tolist() == [0x58, 0x5a, 0, 2, 0x7e, 0x7e, 0x80]
    x = np.random.default_rng(1).standard_normal((130, 200)).astype(np.float32)
    for high in (1, 128):
        stored, scales = cast(x, high)
        assert stored.shape == x.shape and scales.shape == (-(-130 // high), 2)
        assert (np.abs(back(stored, scales, high) - x) <= np.abs(x) * 2.0 ** -4 * 1.001 + scales.max() * 2.0 ** -10).all()
