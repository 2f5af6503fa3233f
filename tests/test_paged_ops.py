"""Descriptors of the operators over a cache in pages: what is refused, and which kernels a call would launch.  No GPU needed."""
import ctypes as C

import pytest

import morello_amd as M
from morello_amd import _binding as B

OK, UNSUPPORTED, BAD_SPEC, NULL, TOO_LARGE = 0, 1, 3, 6, 7


def tables(**given):
    return M.PageTables(**{**dict(requests=4, table_width=8, page_size=16, pages=64, tokens=100, free_pages=20), **given})


def rotary(dtype=M.bf16, **given):
    return M.Rotary(dtype, **{**dict(tokens=33, q_heads=8, kv_heads=2, head_dim=64, sections=[8, 12, 12], page_size=16, pages=9), **given})


def attention(dtype=M.bf16, **given):
    return M.PagedAttention(dtype, **{**dict(tokens=33, requests=4, q_heads=8, kv_heads=2, head_dim=64, page_size=16, pages=64, table_width=8), **given})


def test_struct_sizes_match_the_header():
    assert C.sizeof(B.PageTablesC) == 6 * 4
    assert C.sizeof(B.RotaryC) == 6 * 4 + 4 * 4 + 4 * 4 + (4 * 2 + 2 * 3) * 8
    assert C.sizeof(B.PagedAttentionC) == 12 * 4 + (2 * 2 + 2 * 3) * 8


@pytest.mark.parametrize("given,status", [
    (dict(), OK), (dict(free_pages=0), OK), (dict(page_size=1), OK), (dict(page_size=7), OK),
    (dict(requests=0), BAD_SPEC), (dict(table_width=0), BAD_SPEC), (dict(page_size=0), BAD_SPEC), (dict(pages=0), BAD_SPEC), (dict(tokens=0), BAD_SPEC),
    (dict(pages=1 << 28), TOO_LARGE), (dict(pages=(1 << 27) - 1), OK), (dict(table_width=1 << 27), TOO_LARGE),
    (dict(requests=1 << 29, table_width=4), TOO_LARGE), (dict(tokens=(1 << 23) + 1), TOO_LARGE), (dict(free_pages=1 << 31), TOO_LARGE),
])
def test_page_tables_check(given, status):
    assert tables(**given).check() == status


@pytest.mark.parametrize("given,status", [
    (dict(), OK), (dict(dtype=M.f32), OK), (dict(dtype=M.i8), UNSUPPORTED), (dict(dtype=9), BAD_SPEC), (dict(tokens=0), BAD_SPEC), (dict(q_heads=0), BAD_SPEC),
    (dict(kv_heads=0), BAD_SPEC), (dict(kv_heads=0, page_size=0, pages=0), OK), (dict(head_dim=0), BAD_SPEC), (dict(head_dim=62), BAD_SPEC),
    (dict(sections=[0]), BAD_SPEC), (dict(sections=[32]), OK), (dict(sections=[33]), BAD_SPEC), (dict(sections=[1, 0, 0, 2]), OK),
    (dict(sections=[0xffffffff, 1]), BAD_SPEC), (dict(page_size=0), BAD_SPEC), (dict(page_size=0, pages=0), OK), (dict(pages=0), BAD_SPEC),
    (dict(page_size=1 << 16, pages=1 << 16), TOO_LARGE), (dict(tokens=1 << 24), TOO_LARGE), (dict(q_heads=65536), TOO_LARGE), (dict(head_dim=1 << 24), TOO_LARGE),
    (dict(q_strides=(-1, 64)), BAD_SPEC), (dict(q_strides=(0, 64)), OK), (dict(q_out_strides=(0, 64)), BAD_SPEC), (dict(q_out_strides=(64, 64)), BAD_SPEC),
    (dict(q_out_strides=(512, 64)), OK), (dict(q_out_strides=(64, 33 * 64)), OK), (dict(q_out_strides=(64, 32 * 64)), BAD_SPEC),
    (dict(key_strides=(16 * 128, 128, 64)), OK), (dict(key_strides=(16 * 128, 64, 16 * 64)), OK), (dict(key_strides=(16 * 128 - 1, 128, 64)), BAD_SPEC),
    (dict(value_strides=(16 * 128, 128, 63)), BAD_SPEC), (dict(value_strides=(1 << 41, 128, 64)), BAD_SPEC),
])
def test_rotary_check(given, status):
    assert rotary(**given).check() == status


@pytest.mark.parametrize("given,status", [
    (dict(), OK), (dict(dtype=M.f32), OK), (dict(dtype=M.u8), UNSUPPORTED), (dict(dtype=-1), BAD_SPEC), (dict(tokens=0), BAD_SPEC), (dict(requests=0), BAD_SPEC),
    (dict(q_heads=7), BAD_SPEC), (dict(kv_heads=0), BAD_SPEC), (dict(q_heads=0), BAD_SPEC), (dict(head_dim=1), OK), (dict(head_dim=1024), OK), (dict(head_dim=1025), UNSUPPORTED),
    (dict(page_size=0), BAD_SPEC), (dict(page_size=5), OK), (dict(pages=0), BAD_SPEC), (dict(table_width=0), BAD_SPEC), (dict(table_width=1 << 28), TOO_LARGE),
    (dict(scale=float("nan")), BAD_SPEC), (dict(scale=float("inf")), BAD_SPEC), (dict(scale=-1.0), OK), (dict(window=0xffffffff), OK), (dict(max_new=10 ** 9), OK),
    (dict(out_strides=(64, 64)), BAD_SPEC), (dict(out_strides=(0, 64)), BAD_SPEC), (dict(q_strides=(0, 64)), OK), (dict(key_strides=(0, 0, 64)), OK),
    (dict(key_strides=(64, -64, 64)), BAD_SPEC), (dict(tokens=1 << 24), TOO_LARGE), (dict(requests=1 << 20, table_width=1 << 12), TOO_LARGE),
])
def test_paged_attention_check(given, status):
    op = attention(**given)
    assert op.check() == status
    if status != OK:
        assert op.workspace_bytes() == 0
        with pytest.raises(M.MorelloError) as err:
            op.plan()
        assert err.value.status == status and "(" in str(err.value)


def test_null_descriptors_and_lists():
    lib = B.load()
    for name in ("page_tables", "rotary", "paged_attention"):
        assert getattr(lib, f"mrl_{name}_check")(None) == NULL
        assert getattr(lib, f"mrl_run_{name}")(None, None, None) == NULL
        assert getattr(lib, f"mrl_{name}_plan")(None, None, None, 0) == NULL
    for op in (tables(), rotary(), attention()):
        assert op._run(C.byref(op._c), None, None) == NULL
        with pytest.raises(ValueError):
            op.run_async([1, 2, 3])
    with pytest.raises(ValueError):
        rotary(sections=[1] * 5)
    with pytest.raises(ValueError):
        attention(key_strides=(1, 2))


def test_plans():
    families = set(M.Target.kernels())
    for op in (tables(), rotary(), rotary(M.f32, adjacent=True), attention(), attention(M.f32), attention(head_dim=200), attention(page_size=3)):
        plan = op.plan()
        assert plan.steps and set(plan.kernels) <= families and plan.cost_ns >= 2000 * len(plan.steps), plan
    assert tables(tokens=5000).plan().steps[0].grid[0] == 5
    # 16 bytes at a time, or an element where a stride or a section does not allow that
    assert "V = 8" in rotary(sections=[16, 8, 8]).plan().steps[0].kernel and "V = 1" in rotary(q_strides=(513, 64)).plan().steps[0].kernel
    assert "V = 4" in rotary(M.f32).plan().steps[0].kernel and "V = 1" in rotary(sections=[3]).plan().steps[0].kernel


def test_which_kernels_attention_takes():
    """By the rows that a request may have, the type and what a table holds; strides and sizes that the tiles cannot take go to the generic kernel."""
    steps = lambda **given: [s.kernel.split(" ")[0] for s in attention(**given).plan().steps]
    shared, direct, generic = ["k_paged_attn", "k_paged_attn_merge"], ["k_paged_attn"], ["k_paged_attn_generic"]
    assert steps(max_new=1) == steps(max_new=1, table_width=64) == steps(max_new=1, table_width=32, dtype=M.f32) == direct
    assert steps(max_new=1, table_width=65) == steps(max_new=1, table_width=33, dtype=M.f32) == steps() == steps(dtype=M.f32) == shared
    assert steps(head_dim=136) == steps(head_dim=12) == steps(page_size=24) == steps(q_strides=(516, 64)) == steps(key_strides=(1 << 24, 1 << 24, 64)) == generic
    # a workgroup to a request's head only where that is a launch
    assert steps(max_new=1, requests=1 << 19, q_heads=2) == direct and steps(max_new=1, requests=1 << 20, q_heads=2) == shared
    # places of keys near 2^31
    assert steps(requests=1, table_width=(0x7fff0000 >> 4), pages=64) == shared and steps(requests=1, table_width=(0x7fff0000 >> 4) + 1, pages=64) == generic
    assert attention(max_new=1).workspace_bytes() == 0 and attention(head_dim=136).workspace_bytes() == 0 and attention().workspace_bytes() > 0


@pytest.mark.parametrize("op,given,status", [
    (attention, dict(pages=1 << 23, key_strides=(1 << 40, 128, 64)), TOO_LARGE), (attention, dict(pages=(1 << 27) - 1, value_strides=(1 << 38, 128, 64)), TOO_LARGE),
    (attention, dict(tokens=1 << 23, q_strides=(1 << 40, 64)), TOO_LARGE), (attention, dict(tokens=1 << 23, out_strides=(1 << 40, 64)), TOO_LARGE),
    (attention, dict(pages=1 << 20, key_strides=(1 << 40, 128, 64)), OK), (attention, dict(pages=(1 << 20) + 1, key_strides=(1 << 40, 128, 64)), TOO_LARGE),
    (attention, dict(pages=1 << 26, page_size=2, table_width=64, key_strides=(1 << 33, 1 << 39, 64)), OK), (attention, dict(pages=(1 << 27) - 1, key_strides=(0, 1 << 40, 1 << 40)), OK),
    (rotary, dict(pages=1 << 23, key_strides=(1 << 40, 128, 64)), TOO_LARGE), (rotary, dict(pages=1 << 23, value_strides=(1 << 40, 128, 64)), TOO_LARGE),
    (rotary, dict(pages=1 << 24, page_size=16, key_strides=(1 << 40, 1 << 40, 64)), TOO_LARGE), (rotary, dict(pages=64, page_size=16, key_strides=(1 << 40, 1 << 40, 64)), BAD_SPEC),
    (rotary, dict(tokens=1 << 23, k_strides=(1 << 40, 64)), TOO_LARGE), (rotary, dict(tokens=1 << 23, q_out_strides=(1 << 40, 64)), TOO_LARGE),
    (rotary, dict(tokens=1 << 23, page_size=0, pages=0, key_strides=(0, 1 << 40, 64)), TOO_LARGE), (rotary, dict(pages=1 << 20, key_strides=(1 << 39, 128, 64)), OK),
])
def test_strides_whose_products_pass_63_bits(op, given, status):
    """A stride of 2^40 is legal, and so are 2^27 pages: together their last element has no 64-bit place."""
    assert op(**given).check() == status
