"""Layers of experts for few tokens, against the same in 64 bits."""
import numpy as np
import pytest

import morello_amd as M
from blocks_util import POISON, Device, Layer, as_f64

pytestmark = pytest.mark.gpu

# tokens, hidden, inter, experts, top_k
SIZES = [(1, 256, 128, 8, 2), (1, 1, 1, 1, 1), (1, 2048, 256, 64, 8), (2, 512, 130, 16, 4), (3, 264, 72, 60, 4), (5, 1001, 333, 7, 3), (8, 640, 384, 128, 8), (16, 512, 200, 8, 2),
         (17, 300, 96, 4, 2), (33, 256, 256, 5, 5), (64, 384, 64, 32, 6), (100, 200, 50, 3, 1), (128, 256, 144, 256, 8), (256, 128, 40, 512, 32), (70, 130, 260, 2, 2),
         # logits of all tokens below, at and past the threads that choose; the last that one workgroup chooses for all, and one more
         (5, 264, 72, 60, 4), (2, 128, 64, 127, 5), (2, 128, 64, 128, 5), (3, 128, 64, 104, 7), (16, 136, 40, 45, 3), (32, 64, 48, 32, 4), (31, 64, 48, 32, 16), (33, 64, 48, 31, 4), (1, 64, 48, 181, 32),
         # the largest of whose choices every workgroup makes all, and those behind them
         (8, 72, 40, 32, 32), (8, 72, 40, 33, 32), (4, 136, 64, 64, 6), (1, 136, 64, 181, 32), (1, 136, 64, 182, 32), (32, 64, 48, 8, 2), (28, 64, 48, 9, 2), (29, 64, 48, 9, 2),
         # sixteen waves for the products with down, and one token more
         (64, 300, 136, 128, 8), (65, 300, 136, 128, 8), (64, 2050, 64, 40, 3), (64, 264, 128, 300, 32), (33, 4096, 48, 6, 2), (40, 4100, 48, 64, 2), (1, 5000, 64, 2, 1), (3, 9003, 300, 4, 2), (2, 4096, 48, 8, 2), (5, 2048, 30, 100, 1), (7, 2000, 40, 9, 1), (44, 640, 128, 64, 6), (44, 640, 129, 64, 6), (40, 300, 64, 64, 6), (3, 200, 65, 12, 4),
         # several workgroups to the same rows of down
         (40, 72, 2100, 24, 4), (3, 250, 4000, 8, 3), (128, 65, 900, 16, 4), (1, 1, 8200, 8, 8), (256, 130, 1300, 4, 2)]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", SIZES)
def test_layer(gpu, kind, tokens, hidden, inter, experts, top_k):
    layer = Layer(kind, tokens, hidden, inter, experts, top_k, seed=tokens + hidden, renormalise=bool(tokens % 2))
    layer.check(layer.run())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", [(1, 256, 300, 8, 1), (4, 512, 2100, 16, 4), (3, 2100, 640, 6, 2), (16, 128, 64, 32, 2), (40, 72, 100, 5, 1), (200, 2064, 40, 1, 1), (64, 128, 128, 90, 2)])
def test_small_layers_round_once(gpu, kind, tokens, hidden, inter, experts, top_k):
    """What is between the products in sixteen bits."""
    layer = Layer(kind, tokens, hidden, inter, experts, top_k, seed=21)
    want, bound, _, _ = layer.want(h_step=2.0 ** -16)
    assert (np.abs(as_f64("bf16", layer.run()[0]) - want) <= bound).all()


def test_results_without_bounds(gpu):
    """What is past bf16 between the products, and infinite weights: infinite, not NaN, in one number and in two."""
    for tokens, inter in ((2, 64), (40, 1024)):
        layer = Layer("bf16", tokens, 64, inter, 4, 1, seed=22)
        layer.x &= 0x7fff
        for name in ("gate", "up", "down"):
            layer.stored[name] &= 0x7fff
        layer.stored["up"][:, 3] = 0x7f00   # 1.7e38
        layer.stored["down"][:, 7, 5] = 0x7f80
        layer.x[:] = np.maximum(layer.x, 0x4000)   # (2 and more: 64 such products past 3.4e38)
        assert np.isposinf(as_f64("bf16", layer.run()[0])).all()
        layer.stored["up"][:, 3] = 0
        out = as_f64("bf16", layer.run()[0])
        assert np.isposinf(out[:, 7]).all() and np.isfinite(np.delete(out, 7, 1)).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [-3, 0, 1, 7, 20, 99])
def test_rows_that_count(gpu, kind, rows):
    layer = Layer(kind, 20, 256, 128, 8, 2, seed=3)
    x = layer.x.copy()
    layer.x[max(0, rows):] = POISON["bf16"]   # a padded batch: what lies behind is not read
    got = layer.run(rows=rows)
    layer.x = x
    layer.check(got, rows)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_weights_of_experts_that_nobody_wants_do_not_matter(gpu, kind):
    layer = Layer(kind, 3, 256, 128, 16, 2, seed=5)
    wanted = set(layer.choice()[0].ravel().tolist())
    for e in set(range(16)) - wanted:
        for name in ("gate", "up", "down"):
            layer.stored[name][e] = 0x7f if kind == "e4m3" else POISON["bf16"]
    layer.check(layer.run())


def test_equal_logits_go_to_the_lowest_expert(gpu):
    layer = Layer("bf16", 9, 128, 64, 70, 4, seed=6)
    layer.router[:] = layer.router[3]
    layer.router64[:] = layer.router64[3]
    got = layer.run()
    assert (got[1] == np.arange(4)).all() and (got[2] == np.float32(1 / 70)).all()
    layer.x[:], layer.x64[:] = 0, 0
    got = layer.run()
    assert (got[1] == np.arange(4)).all() and not as_f64("bf16", got[0]).any()


@pytest.mark.parametrize("experts,top_k", [(65, 32), (130, 3), (192, 32), (257, 8), (512, 32), (449, 1), (64, 20)])
def test_choices_among_many(gpu, experts, top_k):
    """Logits with many equals, whole ones: the lowest numbers first, across the sixty-fours that are ranked together; rows of equals, and of the lowest there is."""
    layer = Layer("bf16", 40, 16, 16, experts, top_k, seed=experts)
    layer.x[:], layer.router[:] = 0, 0
    rng = np.random.default_rng(experts)
    layer.x[:, 0] = 0x3f80   # 1
    layer.x[:, 1] = rng.choice([0, 0x3f80, 0xbf80, 0x4000], 40)   # 0, 1, -1, 2
    layer.router[:, :2] = rng.choice([0, 0x3f80, 0x4000, 0x4040, 0xc000], (experts, 2))
    layer.x[0, :2] = 0
    layer.x[1, 0] = 0xff7f   # -3.4e38 times 2 and 3: past 32 bits
    layer.x64, layer.router64 = as_f64("bf16", layer.x), as_f64("bf16", layer.router)
    _, chosen, shares = layer.run()
    want, share = layer.choice()
    assert np.array_equal(chosen, want)
    finite = np.arange(40) != 1
    assert np.allclose(shares[finite], share[finite], rtol=2e-6, atol=1e-38)


@pytest.mark.parametrize("tokens,experts,top_k", [(2, 12, 3), (4, 12, 12), (40, 12, 4), (9, 130, 5)])
@pytest.mark.parametrize("renormalise", [False, True])
def test_logits_out_of_the_range_of_32_bits(gpu, tokens, experts, top_k, renormalise):
    """Products of finite numbers past 3.4e38 and below 1e-45: all different, the later expert's the larger, and shares are numbers."""
    layer = Layer("bf16", tokens, 24, 16, experts, top_k, seed=23, renormalise=renormalise)
    layer.x[:], layer.router[:] = 0, 0
    e = np.arange(experts)
    layer.router[:, 5] = 0x3f80 + e          # 1 and more, up to 2 and more
    layer.router[:, 17] = 0x1f80 + e         # the same times 2^-64
    layer.router[:, 22] = e % 2 * 0x4000     # 2, and nothing
    layer.x[0::2, 5] = 0x7f7f                # 3.4e38
    layer.x[1::2, 17] = 0x1000               # 2^-95: products at 2^-159 and above, where 32 bits have nothing
    layer.x[0, 22] = 0xc0a0                  # -5
    layer.x64, layer.router64 = as_f64("bf16", layer.x), as_f64("bf16", layer.router)
    _, chosen, shares = layer.run()
    want, share = layer.choice()
    assert np.array_equal(want, np.tile(experts - 1 - np.arange(top_k), (tokens, 1)))
    assert np.array_equal(chosen, want)
    assert np.isfinite(shares).all() and np.allclose(shares, share, rtol=2e-6, atol=1e-38)


def test_a_row_that_is_not_a_number(gpu):
    """Its choice is the first experts, its results are NaN, and the other rows are what they are without it."""
    layer = Layer("e4m3", 6, 256, 128, 8, 3, seed=7)
    x = layer.x.copy()
    layer.x[2, 5] = POISON["bf16"]
    out, chosen, shares = layer.run()
    layer.x = x
    assert (chosen[2] == np.arange(3)).all() and np.isnan(shares[2]).all() and np.isnan(as_f64("bf16", out[2])).all()
    want, bound, which, _ = layer.want()
    others = np.arange(6) != 2
    assert np.array_equal(chosen[others], which[others]) and (np.abs(as_f64("bf16", out) - want) <= bound)[others].all()


@pytest.mark.parametrize("hidden,inter", [(64, 300), (64, 129), (2050, 300), (64, 384)])
def test_an_unbounded_scale_of_the_last_block(gpu, hidden, inter):
    """Is that block's alone: with all else positive every element of the result is infinite, not NaN from what would lie behind it."""
    layer = Layer("e4m3", 3, hidden, inter, 4, 1, seed=9)
    layer.x &= 0x7fff
    for name in ("gate", "up", "down"):
        layer.stored[name] = layer.stored[name] & 0x3f | 0x20   # 2^-3 to 1.875
    layer.scales["down"][:, :, -1] = np.inf
    assert np.isposinf(as_f64("bf16", layer.run()[0])).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_strides_and_odd_addresses(gpu, kind):
    """gate and up behind each other in one stack, rows with gaps of NaN, and all of it off 16 bytes."""
    layer = Layer(kind, 11, 264, 128, 6, 2, seed=8)
    size = np.uint8 if kind == "e4m3" else np.uint16
    poison = 0x7f if kind == "e4m3" else POISON["bf16"]
    for gap, shift in ((0, 0), (8, 0), (3, 1)):
        row = layer.hidden + gap
        both = np.full(shift + 6 * 2 * 128 * row, poison, size)
        stack = both[shift:].reshape(6, 2, 128, row)
        stack[:, 0, :, :layer.hidden], stack[:, 1, :, :layer.hidden] = layer.stored["gate"], layer.stored["up"]
        down_row = layer.inter + gap
        down = np.full(shift + 6 * layer.hidden * down_row, poison, size)
        down[shift:].reshape(6, layer.hidden, down_row)[:, :, :layer.inter] = layer.stored["down"]
        x = np.full((11, row), POISON["bf16"], np.uint16)
        x[:, :layer.hidden] = layer.x
        out = np.full((11, row), POISON["bf16"], np.uint16)
        given = dict(gate_strides=(2 * 128 * row, row), up_strides=(2 * 128 * row, row), down_strides=(layer.hidden * down_row, down_row), x_stride=row, out_stride=row)
        scales = [None, None, None]
        if kind == "e4m3":
            blocks = layer.scales["gate"].shape[2]
            given.update(gate_scale_strides=(2 * blocks, blocks), up_scale_strides=(2 * blocks, blocks))
            scales = [np.stack([layer.scales["gate"], layer.scales["up"]], 1), None, layer.scales["down"]]
        op = layer.op(**given)
        with Device() as d:
            stack_at = d.put(both, shift)
            item = both.itemsize
            pointers = [d.put(x), d.put(layer.router), stack_at, stack_at + 128 * row * item, d.put(down, shift)]
            if kind == "e4m3":
                s = d.put(scales[0])
                pointers += [s, s + 4 * layer.scales["gate"].shape[2], d.put(scales[2])]
            else:
                pointers += [None, None, None]
            pointers.append(None)
            at = len(d.bufs)
            pointers += [d.put(out), None, None, d.put(np.full(max(16, op.workspace_bytes()), 0xff, np.uint8))]
            op.run_device(pointers)
            got = d.get(at, out)
        assert (got[:, layer.hidden:] == POISON["bf16"]).all()
        want, bound, _, _ = layer.want()
        assert (np.abs(as_f64("bf16", got[:, :layer.hidden]) - want) <= bound).all(), (gap, shift)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_repeats_bit_for_bit(gpu, kind):
    layer = Layer(kind, 40, 512, 256, 16, 4, seed=9)
    first = layer.run()
    second = layer.run()
    assert all(np.array_equal(a, b) for a, b in zip(first, second))


# Sixteen rows of down at a time, in several turns and in one, of tokens that one workgroup has all of and that several share; rows of all ends; eight rows off and on steps of 256 bytes
MORE = [(64, 4112, 256, 8, 2), (20, 2100, 300, 6, 2), (256, 2100, 140, 8, 2), (256, 2056, 7, 16, 8), (256, 64, 7, 16, 8), (35, 2112, 512, 6, 1), (35, 2100, 500, 6, 1), (80, 2056, 7, 430, 32),
        (80, 64, 7, 430, 32), (40, 200, 64, 64, 8), (90, 200, 40, 80, 5), (12, 320, 1536, 16, 4), (32, 1800, 256, 24, 3), (35, 4200, 512, 6, 1), (3, 2100, 256, 4, 2), (2, 2056, 5, 4, 2),
        (256, 7, 64, 16, 8), (33, 4100, 48, 6, 2), (40, 5, 40, 64, 2)]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", MORE)
def test_more_layers(gpu, kind, tokens, hidden, inter, experts, top_k):
    layer = Layer(kind, tokens, hidden, inter, experts, top_k, seed=tokens + hidden, renormalise=bool(tokens % 2))
    first = layer.run()
    layer.check(first)
    assert all(np.array_equal(a, b) for a, b in zip(first, layer.run()))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", [
    (5, 256, 640, 4, 2), (9, 520, 1100, 12, 3), (16, 2100, 700, 6, 2), (32, 384, 768, 32, 8), (33, 300, 520, 5, 5), (64, 1030, 256, 8, 2), (100, 200, 333, 7, 3), (130, 2064, 200, 4, 2), (256, 128, 130, 16, 4)])
def test_all_layers_round_once(gpu, kind, tokens, hidden, inter, experts, top_k):
    """What is between the products in sixteen bits whatever the sizes, many tokens of each expert and few: errors are those of the result's own rounding, spread evenly over a step, whose mean square is a twelfth of the
    step's.  Of 1280 elements and more that mean is good to 3 %; a tenth more of its root is allowed, where sixteen bits add a ten thousandth and eight bits four tenths."""
    layer = Layer(kind, tokens, hidden, inter, experts, top_k, seed=24)
    want, bound, _, _ = layer.want(h_step=2.0 ** -16)
    off = as_f64("bf16", layer.run()[0]) - want
    assert (np.abs(off) <= bound).all(), f"{(np.abs(off) / bound).max():.2f} of the bound"
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(want), 2.0 ** -100))) - 7)
    assert np.mean(off ** 2) <= 1.1 ** 2 * np.mean(step ** 2 / 12)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_token_among_others_and_alone(gpu, kind):
    """Its result is the same but for the order of sums in 32 bits, whose errors, some 2^-20 of a result, turn the rounding to bf16 of one element in thousands: less than one in twenty."""
    layer = Layer(kind, 48, 384, 300, 6, 2, seed=25)
    among = as_f64("bf16", layer.run()[0])
    _, bound, _, _ = layer.want(h_step=2.0 ** -16)
    one = Layer(kind, 1, 384, 300, 6, 2, seed=25)
    one.router, one.stored, one.scales = layer.router, layer.stored, layer.scales
    for t in (0, 17, 47):
        one.x = layer.x[t:t + 1].copy()
        alone = as_f64("bf16", one.run()[0])[0]
        assert (np.abs(among[t] - alone) <= 2 * bound[t]).all() and (among[t] != alone).mean() < 0.05
