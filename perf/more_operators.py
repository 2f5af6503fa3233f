"""Feed-forward layers on weights in 8 bits, as a serving program runs them, for timing and for comparing results.

Weights and activations go to e4m3 with a scale for each block of 128 (`M.CastBlocks`: weights once, in blocks of 128 x 128,
activations before each product, in blocks of 1 x 128, behind the gate of a gated layer where there is one); dense layers are products
of two such tensors (`M.MatmulBlocks`); a layer of experts routes a few tokens to their experts and runs those (`M.Experts`).  The
listed cases go from a decoding step of one token to prompts of thousands; `draw` gives further sizes, types and layouts of the same kinds of work.
"""
import math

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4, "e4m3": 1}
_LEAST = 2.0 ** -110  # a block's largest value counts as at least this much


def _cast(dtype, rows, cols, block_rows=1, gated=False):
    return {"op": "cast", "dtype": dtype, "rows": rows, "cols": cols, "block_rows": block_rows, "gated": gated}


def _product(out, m, n, k):
    return {"op": "product", "out": out, "m": m, "n": n, "k": k}


def _experts(weights, tokens, hidden, inter, experts, top_k, renormalise=False):
    return {"op": "experts", "weights": weights, "tokens": tokens, "hidden": hidden, "inter": inter, "experts": experts, "top_k": top_k,
            "renormalise": renormalise}


def listed():
    return [
        # A decoding step's activations before a product: all latency.
        dict(_cast("bf16", 16, 4096), name="cast_decode"),
        # A long prompt's between the two products of a gated layer.
        dict(_cast("bf16", 4101, 8192, gated=True), name="cast_gated_prompt"),
        # A layer's weights as a checkpoint holds them, rows and columns that do not fill their blocks.
        dict(_cast("f32", 8100, 4110, block_rows=128), name="cast_weights"),
        # A decoding step of a small batch through a dense layer: the weights are read once.
        dict(_product("bf16", 8, 4096, 4096), name="product_decode"),
        # A larger batch with drafted tokens.
        dict(_product("bf16", 67, 6144, 4096), name="product_batch"),
        # A prompt's chunk.
        dict(_product("bf16", 4096, 4096, 4096), name="product_prompt"),
        # Prompts together through a wide layer: the largest.
        dict(_product("bf16", 8192, 8192, 8192), name="product_large"),
        # Sizes that no tile divides, sums kept in f32.
        dict(_product("f32", 1001, 2050, 4425), name="product_odd"),
        # One token through a layer of small experts.
        dict(_experts("bf16", 1, 2048, 1024, 64, 8), name="experts_one"),
        # A decoding batch through many small experts in 8 bits: most of them are wanted.
        dict(_experts("e4m3", 32, 2048, 768, 128, 8, renormalise=True), name="experts_batch"),
        # A batch through few large experts: all of them are wanted.
        dict(_experts("bf16", 16, 4096, 14336, 8, 2, renormalise=True), name="experts_wide"),
        # Sizes that no block or tile divides.
        dict(_experts("e4m3", 5, 2056, 1416, 60, 4), name="experts_odd"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _near(rng, lo, hi, step):
    """A multiple of `step`, or one time in five any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.2 else max(1, round(n / step)) * step


def draw(rng):
    kind = rng.choice(["cast", "product", "product", "experts", "experts"])
    if kind == "cast":
        if rng.random() < 0.25:
            return _cast(rng.choice(["bf16", "f32"]), _near(rng, 128, 8192, 128), _near(rng, 128, 4096, 128), block_rows=128)
        return _cast(rng.choice(["bf16", "bf16", "f32"]), _log(rng, 1, 4096), _near(rng, 64, 8192, 64), gated=rng.random() < 0.5)
    if kind == "product":
        m = rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192), _near(rng, 64, 8192, 64)])
        return _product(rng.choice(["bf16", "bf16", "f32"]), m, _near(rng, 128, 8192, 64), _near(rng, 128, 8192, 128))
    experts, top_k = rng.choice([(8, 2), (16, 4), (60, 4), (64, 6), (64, 8), (128, 8), (256, 8)])
    hidden = _near(rng, 256, 7168, 64)
    inter = _near(rng, 64, min(14336, max(65, int(1.2e9 / (experts * hidden)))), 64)
    return _experts(rng.choice(["bf16", "e4m3", "e4m3"]), rng.choice([1, _log(rng, 1, 128), _log(rng, 1, 32)]), hidden, inter, experts, top_k, rng.random() < 0.5)


def _spread_amax(x, block_rows):
    """The largest size of each block of block_rows x 128 of a matrix, or of each of a stack."""
    rows, cols = x.shape[-2:]
    padded = torch.nn.functional.pad(x.abs(), (0, -cols % 128, 0, -rows % block_rows))
    return padded.unflatten(-1, (-1, 128)).unflatten(-3, (-1, block_rows)).amax((-1, -3))


def _over_blocks(scales, rows, cols, block_rows):
    """A scale for each element."""
    return scales.repeat_interleave(block_rows, -2)[..., :rows, :].repeat_interleave(128, -1)[..., :cols]


def _to_blocks(x, block_rows):
    """x, in 32 bits -> (e4m3, scales): the largest of a block comes to 448, the type's largest."""
    amax = _spread_amax(x, block_rows).clamp(min=_LEAST)
    scales, factors = amax / 448.0, 448.0 / amax
    return (x * _over_blocks(factors, *x.shape[-2:], block_rows)).to(torch.float8_e4m3fn), scales


def _from_blocks(values, scales, block_rows):
    return values.float() * _over_blocks(scales, *values.shape[-2:], block_rows)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std

    def activations(rows, cols):
        """Normal, a few columns many times as large as the others."""
        x = normal(rows, cols)
        wide = torch.randint(cols, (max(1, cols // 256),), generator=gen, device="cuda")
        x[:, wide] *= 20.0
        return x

    def zeros(*shape, dtype):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    state = {"case": case, "call": None}
    if case["op"] == "cast":
        rows, cols, high = case["rows"], case["cols"], case["block_rows"]
        x = activations(rows, 2 * cols if case["gated"] else cols) if high == 1 else normal(rows, cols, std=cols ** -0.5)
        state.update(x=x.to(_TORCH[case["dtype"]]), out=zeros(rows, cols, dtype=torch.uint8), scales=zeros(-(-rows // high), -(-cols // 128), dtype=torch.float32))
        return state
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        state["a"], state["a_scales"] = _to_blocks(activations(m, k), 1)
        state["b"], state["b_scales"] = _to_blocks(normal(n, k, std=k ** -0.5), 128)
        state["out"] = zeros(m, n, dtype=_TORCH[case["out"]])
        return state
    tokens, hidden, inter, experts = case["tokens"], case["hidden"], case["inter"], case["experts"]
    state["x"] = normal(tokens, hidden).to(torch.bfloat16)
    state["router"] = normal(experts, hidden, std=1.5 * hidden ** -0.5).to(torch.bfloat16)  # logits of a standard deviation of 1.5
    for name, rows, cols in (("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter)):
        size = 1 if case["weights"] == "e4m3" else 2
        state[name] = zeros(experts, rows, cols * size, dtype=torch.uint8).view(torch.float8_e4m3fn if size == 1 else torch.bfloat16)
        if size == 1:
            state[name + "_scales"] = zeros(experts, -(-rows // 128), -(-cols // 128), dtype=torch.float32)
        for e in range(experts):
            w = normal(rows, cols, std=cols ** -0.5)
            if size == 1:
                values, scales = _to_blocks(w, 128)
                state[name][e], state[name + "_scales"][e] = values, scales
            else:
                state[name][e] = w
    state["out"] = zeros(tokens, hidden, dtype=torch.bfloat16)
    state["chosen"], state["shares"] = zeros(tokens, case["top_k"], dtype=torch.int32), zeros(tokens, case["top_k"], dtype=torch.float32)
    return state


def run(state):
    if own:
        return _run_own(state)
    return {"cast": _plain_cast, "product": _plain_product, "experts": _plain_experts}[state["case"]["op"]](state)


def _run_own(s):
    """What a program keeps per layer: the descriptor and the pointers of its buffers."""
    case = s["case"]
    if s["call"] is None:
        import morello_amd as M

        M.init(0)
        types = {"bf16": M.bf16, "f32": M.f32, "e4m3": M.f8e4m3}
        if case["op"] == "cast":
            op = M.CastBlocks(types[case["dtype"]], rows=case["rows"], cols=case["cols"], block_rows=case["block_rows"], gated=case["gated"])
            names = ("x", "out", "scales")
        elif case["op"] == "product":
            op = M.MatmulBlocks(types[case["out"]], m=case["m"], n=case["n"], k=case["k"])
            names = ("a", "a_scales", "b", "b_scales", "out", "workspace")
        else:
            op = M.Experts(types[case["weights"]], tokens=case["tokens"], hidden=case["hidden"], inter=case["inter"], experts=case["experts"],
                           top_k=case["top_k"], renormalise=case["renormalise"])
            names = ("x", "router", "gate", "up", "down", "gate_scales", "up_scales", "down_scales", "rows", "out", "chosen", "shares", "workspace")
        if case["op"] != "cast":
            s["workspace"] = torch.zeros(max(1, op.workspace_bytes()), dtype=torch.uint8, device="cuda")
        s["call"] = (op, [s[n].data_ptr() if n in s else 0 for n in names])
    op, pointers = s["call"]
    op.run_async(pointers, torch.cuda.current_stream().cuda_stream)
    if case["op"] == "cast":
        return [s["out"].view(torch.float8_e4m3fn), s["scales"]]
    return s["out"] if case["op"] == "product" else [s["out"], s["chosen"], s["shares"]]


def _plain_cast(s):
    x = s["x"].float()
    if s["case"]["gated"]:
        gate, up = x.chunk(2, -1)
        x = gate / (1.0 + torch.exp(-gate)) * up
    return list(_to_blocks(x, s["case"]["block_rows"]))


def _plain_product(s):
    a = _from_blocks(s["a"], s["a_scales"], 1)
    return torch.mm(a, _from_blocks(s["b"], s["b_scales"], 128).t()).to(s["out"].dtype)


def _plain_experts(s):
    """The experts of each token where those are few, or all experts on all tokens, those that a token did not choose with a share of nothing."""
    case = s["case"]
    x, experts, top_k = s["x"].float(), case["experts"], case["top_k"]
    probabilities = torch.softmax(s["x"].double() @ s["router"].double().t(), -1)
    order = torch.sort(probabilities, dim=-1, descending=True, stable=True)
    chosen, shares = order.indices[:, :top_k], order.values[:, :top_k]
    if case["renormalise"]:
        shares = shares / shares.sum(-1, keepdim=True)
    few = chosen.numel() <= experts
    wanted = chosen.flatten() if few else slice(None)

    def weights(name):
        w = s[name]
        if case["weights"] == "e4m3":
            return _from_blocks(w.view(torch.uint8)[wanted].view(w.dtype), s[name + "_scales"][wanted], 128)
        return w[wanted].float()

    def product(w):
        return torch.bmm(w, x.repeat_interleave(top_k, 0)[:, :, None]) if few else torch.mm(w.flatten(0, 1), x.t()).view(experts, case["inter"], -1)

    gate, up = product(weights("gate")), product(weights("up"))
    each = torch.bmm(weights("down"), (gate / (1.0 + torch.exp(-gate)) * up).contiguous())  # a choice, or an expert; hidden; a token each
    if few:
        out = (each.view(-1, top_k, case["hidden"]) * shares.float()[:, :, None]).sum(1)
    else:
        dense = torch.zeros_like(probabilities).scatter(1, chosen, shares).float()
        out = (each * dense.t()[:, None, :]).sum(0).t()
    return [out.to(torch.bfloat16), chosen.to(torch.int32), shares.float()]


def _e4m3(x):
    """x in 64 bits, rounded to the nearest number of four bits from 2^-6 on and of steps of 2^-9 below, ties to even."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _wide(values, scales, high):
    """Values of blocks in 64 bits, block after block."""
    wide = values.double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            wide[i * high:(i + 1) * high, j * 128:(j + 1) * 128] *= scales[i, j].double()
    return wide


def _rows_wide(values, scales):
    wide = values.double()
    for j in range(scales.shape[1]):
        wide[:, j * 128:(j + 1) * 128] *= scales[:, j:j + 1].double()
    return wide


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cast":
        x, high, cols = s["x"].double(), case["block_rows"], case["cols"]
        if case["gated"]:
            x = x[:, :cols] * torch.sigmoid(x[:, :cols]) * x[:, cols:]
        out, scales = torch.empty_like(x), torch.empty(s["scales"].shape, dtype=torch.float64, device="cuda")
        for j in range(scales.shape[1]):
            part = x[:, j * 128:(j + 1) * 128]
            largest = part.abs().amax(1)
            for i in range(scales.shape[0] if high > 1 else 1):
                rows = slice(i * high, (i + 1) * high) if high > 1 else slice(None)
                scale = (largest[rows].max() if high > 1 else largest).clamp(min=_LEAST) / 448.0
                scales[i if high > 1 else slice(None), j] = scale
                out[rows, j * 128:(j + 1) * 128] = _e4m3(part[rows] / (scale if high > 1 else scale[:, None]))
        return [out, scales]
    if case["op"] == "product":
        if 2.0 * case["m"] * case["n"] * case["k"] > 2e11:
            return None
        return _rows_wide(s["a"], s["a_scales"]) @ _wide(s["b"], s["b_scales"], 128).t()
    tokens, top_k = case["tokens"], case["top_k"]
    x = s["x"].double()
    logits = (x[:, None, :] * s["router"].double()).sum(-1)
    shares = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
    weight, chosen = shares.topk(top_k, -1)
    if case["renormalise"]:
        weight = weight / weight.sum(-1, keepdim=True)
    out = torch.zeros(tokens, case["hidden"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        rows, place = (chosen == e).nonzero(as_tuple=True)
        if rows.numel() == 0:
            continue
        gate, up, down = (_wide(s[n][e], s[n + "_scales"][e], 128) if case["weights"] == "e4m3" else s[n][e].double() for n in ("gate", "up", "down"))
        g = x[rows] @ gate.t()
        out.index_add_(0, rows, weight[rows, place, None] * ((g * torch.sigmoid(g) * (x[rows] @ up.t())) @ down.t()))
    return [out, None, weight]


def work(case):
    if case["op"] == "cast":
        rows, cols = case["rows"], case["cols"]
        read = rows * cols * (2 if case["gated"] else 1) * _SIZE[case["dtype"]]
        return {"bytes": read + rows * cols + 4 * -(-rows // case["block_rows"]) * -(-cols // 128), "flops": (7 if case["gated"] else 2) * rows * cols}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = -(-k // 128) * (m + -(-n // 128))
        return {"bytes": (m + n) * k + 4 * scales + m * n * _SIZE[case["out"]], "flops": 2 * m * n * k}
    tokens, hidden, inter, experts, top_k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))
    wanted = experts * (1 - (1 - top_k / experts) ** tokens)  # experts that some token chooses, where they choose alike
    weights = 3 * inter * hidden * _SIZE[case["weights"]] * (1 + 4 / 16384 if case["weights"] == "e4m3" else 1)
    return {"bytes": int(wanted * weights) + 2 * experts * hidden + 4 * tokens * hidden + 8 * tokens * top_k,
            "flops": 2 * tokens * (3 * top_k * inter * hidden + experts * hidden)}
