"""Feed-forward layers as a serving program runs them: activations to e4m3, products, the gate, a layer of experts behind a step's page tables; eager, recorded into
graphs that are replayed while inputs and rows change, side by side on two streams."""
import ctypes as C

import numpy as np
import pytest

import morello_amd as M
from blocks_util import HALF_STEP, POISON, Device, Layer, as_f64, back, cast, over_blocks, product_bound, values
from morello_amd import _binding as B
from morello_amd import synth
from test_gpu_graph_capture import hip_runtime
from test_gpu_paged_step import Recorded, same

pytestmark = pytest.mark.gpu

REQUESTS, PAGE, WIDTH = 4, 16, 8


class Program:
    """A dense gated layer in e4m3 over a step's rows, then a layer of experts over as many of them as the step's requests have new tokens for."""

    def __init__(self, tokens, hidden, inter, kind, seed):
        self.tokens, self.hidden, self.inter, self.seed = tokens, hidden, inter, seed
        self.layer = Layer(kind, tokens, hidden, 200, 12, 3, seed)
        self.ops = {
            "tables": M.PageTables(REQUESTS, WIDTH, PAGE, 40, tokens, 40),
            "cast": M.CastBlocks(M.bf16, tokens, hidden), "both": M.MatmulBlocks(M.bf16, tokens, 2 * inter, hidden),
            "gated": M.CastBlocks(M.bf16, tokens, inter, gated=True), "down": M.MatmulBlocks(M.bf16, tokens, hidden, inter), "experts": self.layer.op()}
        blocks = lambda n: -(-n // 128)
        host = {"x": np.zeros((tokens, hidden), np.uint16), "x8": np.zeros((tokens, hidden), np.uint8), "xs": np.zeros((tokens, blocks(hidden)), np.float32),
                "gu": np.zeros((tokens, 2 * inter), np.uint16), "h8": np.zeros((tokens, inter), np.uint8), "hs": np.zeros((tokens, blocks(inter)), np.float32),
                "y": np.zeros((tokens, hidden), np.uint16), "out": np.full((tokens, hidden), POISON["bf16"], np.uint16),
                "chosen": np.zeros((tokens, 3), np.int32), "shares": np.zeros((tokens, 3), np.float32), "router": self.layer.router,
                "cached": np.zeros(REQUESTS, np.int32), "added": np.zeros(REQUESTS, np.int32), "free": np.arange(40, dtype=np.int32), "count": np.array([40], np.int32),
                "table": np.full((REQUESTS, WIDTH), -1, np.int32), "starts": np.zeros(REQUESTS + 1, np.int32), "lengths": np.zeros(REQUESTS, np.int32),
                "slots": np.zeros(tokens, np.int32), "positions": np.zeros(tokens, np.int32), "left": np.zeros(2, np.int32)}
        for i, (name, rows, cols) in enumerate((("wgu", 2 * inter, hidden), ("wd", hidden, inter))):
            host[name], host[name + "s"] = cast((synth.normal_f32(seed, 10 + i, (rows, cols)) * cols ** -0.5).astype(np.float32), 128)
        for name in ("gate", "up", "down"):
            host["e_" + name] = self.layer.stored[name]
            host["s_" + name] = self.layer.scales.get(name, np.zeros(1, np.float32))
        for name in ("both", "down", "experts"):
            host["w_" + name] = np.full(max(16, self.ops[name].workspace_bytes()), 0xff, np.uint8)
        self.host, self.buffers = host, {n: M.DeviceBuffer.from_numpy(a) for n, a in host.items()}

    def upload(self, name, array):
        array = np.ascontiguousarray(array, self.host[name].dtype)
        assert array.shape == self.host[name].shape
        M._check(B.load().mrl_memcpy_h2d(self.buffers[name].ptr, array.ctypes.data, array.nbytes), "mrl_memcpy_h2d")
        self.host[name] = array

    def read(self, name):
        return self.buffers[name].to_numpy(self.host[name].dtype, self.host[name].shape)

    def inputs(self, step, added):
        self.upload("x", values("bf16", self.seed + step, 20, (self.tokens, self.hidden))[0])
        self.upload("added", added)
        self.upload("out", np.full((self.tokens, self.hidden), POISON["bf16"], np.uint16))

    def enqueue(self, stream):
        p = {n: b.ptr for n, b in self.buffers.items()}
        run = lambda op, *names: self.ops[op].run_async([n if n is None or isinstance(n, int) else p[n] for n in names], stream)
        run("tables", "cached", "added", "free", "count", "table", "starts", "lengths", "slots", "positions", "left")
        run("cast", "x", "x8", "xs")
        run("both", "x8", "xs", "wgu", "wgus", "gu", "w_both")
        run("gated", "gu", "h8", "hs")
        run("down", "h8", "hs", "wd", "wds", "y", "w_down")
        run("experts", "y", "router", "e_gate", "e_up", "e_down", "s_gate", "s_up", "s_down", p["starts"] + 4 * REQUESTS, "out", "chosen", "shares", "w_experts")

    def results(self):
        return {n: self.read(n) for n in ("x8", "xs", "gu", "h8", "hs", "y", "out", "starts")}

    def check(self):
        """Each stage from what the one before left."""
        h, got = self.host, self.results()
        x8, xs = cast(as_f64("bf16", h["x"]), 1)
        assert np.array_equal(got["x8"], x8) and np.array_equal(got["xs"], xs)
        for name, a, a_s, w, out in (("both", "x8", "xs", "wgu", "gu"), ("down", "h8", "hs", "wd", "y")):
            a64, b64 = back(got[a], got[a_s], 1), back(h[w], h[w + "s"], 128)
            want = a64 @ b64.T
            off = np.abs(as_f64("bf16", got[out]) - want)
            assert (off <= product_bound(a64, b64, a64.shape[1] // 128 + 1, HALF_STEP["bf16"], want, cut=True)).all(), name
        g, u = (as_f64("bf16", x) for x in np.split(got["gu"], 2, 1))
        y = g / (1 + np.exp(-g)) * u
        s = over_blocks(got["hs"].astype(np.float64), *y.shape, 1)
        assert (np.abs(back(got["h8"], got["hs"], 1) - y) <= np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10) * 1.001).all()
        rows = int(got["starts"][-1])
        assert rows == int(np.sum(h["added"]))
        self.layer.x, self.layer.x64 = got["y"], as_f64("bf16", got["y"])
        want, bound, _, _ = self.layer.want(rows)
        assert (np.abs(as_f64("bf16", got["out"][:rows]) - want) <= bound).all()
        assert (got["out"][rows:] == POISON["bf16"]).all(), "rows behind the last token were written"

    def free(self):
        for b in self.buffers.values():
            b.free()


STEPS = [[20, 1, 0, 9], [1, 1, 1, 1], [0, 0, 0, 0], [3, 0, 17, 20], [1, 1, 0, 1]]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_steps_of_a_program(gpu, kind):
    stream = M.Stream()
    program = Program(40, 384, 300, kind, seed=51)
    for step, added in enumerate(STEPS):
        program.inputs(step, added)
        program.enqueue(stream)
        stream.synchronize()
        program.check()
    program.free()
    stream.destroy()


@pytest.mark.parametrize("tokens,hidden,inter,kind", [(40, 384, 300, "e4m3"), (200, 512, 640, "bf16")])
def test_graphs_replayed_while_rows_change(gpu, tokens, hidden, inter, kind):
    """Two recorded programs side by side on streams and workspaces of their own, and the same steps run eagerly between their replays."""
    hip = hip_runtime()
    recorded, eager = [Program(tokens, hidden, inter, kind, s) for s in (52, 53)], [Program(tokens, hidden, inter, kind, s) for s in (52, 53)]
    streams = [M.Stream(), M.Stream()]
    graphs = [Recorded(hip, p, s) for p, s in zip(recorded, streams)]
    for step, added in enumerate(STEPS):
        for p in recorded + eager:
            p.inputs(step, added)
        for g, s in zip(graphs, streams):
            g.launch(s)
        for p in eager:
            p.enqueue(None)
        M.synchronize()
        for s in streams:
            s.synchronize()
        for r, e in zip(recorded, eager):
            assert same(r.results(), e.results()), step
    eager[0].check()
    for g in graphs:
        g.destroy()
    for p in recorded + eager:
        p.free()
    for s in streams:
        s.destroy()


def test_a_workspace_that_two_recordings_share(gpu):
    """Launched one after the other on a stream, two recordings may have the same workspace: nothing of a call is left for the next."""
    hip = hip_runtime()
    stream = M.Stream()
    a, b = (Layer("e4m3", 30, 256, 128, 40, 4, seed) for seed in (61, 62))
    alone = [x.run() for x in (a, b)]
    ops = [x.op() for x in (a, b)]
    shared = M.DeviceBuffer.from_numpy(np.full(max(o.workspace_bytes() for o in ops), 0xff, np.uint8))
    with Device() as d:
        pointers, outs = [], []
        for x in (a, b):
            arrays = x.arrays()
            pointers.append([None if y is None else d.put(y) for y in arrays] + [shared.ptr])
            outs.append((pointers[-1][9], arrays[9]))

        class One:
            def __init__(self, i):
                self.i = i

            def enqueue(self, s):
                ops[self.i].run_async(pointers[self.i], s)

        graphs = [Recorded(hip, One(i), stream) for i in (0, 1)]
        for i in (0, 1, 1, 0, 1, 0, 0):
            graphs[i].launch(stream)
            stream.synchronize()
            got = np.empty_like(outs[i][1])
            M._check(B.load().mrl_memcpy_d2h(got.ctypes.data, outs[i][0], got.nbytes), "mrl_memcpy_d2h")
            assert np.array_equal(got, alone[i][0])
        for g in graphs:
            g.destroy()
    shared.free()
    stream.destroy()


def test_sums_that_workgroups_share_in_graphs(gpu):
    """A product and a layer whose sums meet in the workspace, recorded, replayed with other inputs and other rows between eager calls on workspaces full of NaN."""
    hip = hip_runtime()
    stream = M.Stream()
    m, n, k = 130, 200, 5000
    product, layer = M.MatmulBlocks(M.bf16, m, n, k), Layer("e4m3", 20, 64, 4000, 8, 2, seed=71)
    experts = layer.op()
    families = [s.family for op in (product, experts) for s in op.plan().steps]
    assert "k_product_join" in families and "k_experts_join" in families
    b8, b_scales = cast((synth.normal_f32(72, 0, (n, k)) * k ** -0.5).astype(np.float32), 128)
    with Device() as d:
        arrays = layer.arrays()
        arrays[8] = np.array([20], np.int32)
        at = [None if y is None else d.put(y) for y in arrays]
        a8, a_scales = cast(synth.normal_f32(73, 0, (m, k)).astype(np.float32), 1)
        fixed = [d.put(x) for x in (a8, a_scales, b8, b_scales)]
        results = []
        for _ in range(2):   # of the graph, of eager calls
            results.append([d.put(np.zeros((m, n), np.uint16)), d.put(np.full((20, 64), POISON["bf16"], np.uint16))]
                           + [d.put(np.full(op.workspace_bytes(), 0xff, np.uint8)) for op in (product, experts)])

        def calls(where, s):
            out, y, w0, w1 = results[where]
            product.run_async(fixed + [out, w0], s)
            experts.run_async(at[:9] + [y, at[10], at[11], w1], s)

        class Calls:
            enqueue = staticmethod(lambda s: calls(0, s))

        lib = B.load()

        def get(p, shape):
            got = np.empty(shape, np.uint16)
            M._check(lib.mrl_memcpy_d2h(got.ctypes.data, p, got.nbytes), "mrl_memcpy_d2h")
            return got

        def put(p, x):
            M._check(lib.mrl_memcpy_h2d(p, np.ascontiguousarray(x).ctypes.data, x.nbytes), "mrl_memcpy_h2d")

        graph = Recorded(hip, Calls, stream)
        for i, rows in enumerate((20, 7, 0, 1, 20)):
            a8, a_scales = cast(synth.normal_f32(74 + i, 0, (m, k)).astype(np.float32), 1)
            x = values("bf16", 80 + i, 0, (20, 64))[0]
            for p, y in ((fixed[0], a8), (fixed[1], a_scales), (at[0], x), (at[8], np.array([rows], np.int32))):
                put(p, y)
            for r in results:
                put(r[1], np.full((20, 64), POISON["bf16"], np.uint16))
            graph.launch(stream)
            calls(1, None)
            stream.synchronize()
            M.synchronize()
            assert np.array_equal(get(results[0][0], (m, n)), get(results[1][0], (m, n))) and np.array_equal(get(results[0][1], (20, 64)), get(results[1][1], (20, 64)))
            a64, b64 = back(a8, a_scales, 1), back(b8, b_scales, 128)
            want = a64 @ b64.T
            assert (np.abs(as_f64("bf16", get(results[0][0], (m, n))) - want) <= product_bound(a64, b64, 41, HALF_STEP["bf16"], want, cut=True)).all()
            layer.x, layer.x64 = x, as_f64("bf16", x)
            want, bound, _, _ = layer.want(rows)
            got = get(results[0][1], (20, 64))
            assert (np.abs(as_f64("bf16", got[:rows]) - want) <= bound).all() and (got[rows:] == POISON["bf16"]).all()
        graph.destroy()
    stream.destroy()


def test_refusals_of_a_run(gpu):
    """What only a run can see: missing pointers, workspaces off 16 bytes; nothing is launched."""
    layer = Layer("e4m3", 2, 128, 64, 4, 2, seed=7)
    op = layer.op()
    lib = B.load()
    with Device() as d:
        buf = d.put(np.zeros(1 << 16, np.uint8))
        before = M.launch_count()
        run = lambda o, p: o._run(C.byref(o._c), o._pack(*p), None)
        full = [buf] * 13
        for i in (0, 1, 2, 3, 4, 5, 6, 7, 9, 12):
            assert run(op, full[:i] + [0] + full[i + 1:]) == 6, i
        assert run(op, full[:12] + [buf + 8]) == 1
        product = M.MatmulBlocks(M.bf16, 40, 40, 100)   # (rows off 16 bytes: a workspace for their copies)
        assert product.workspace_bytes() > 0
        for i in range(6):
            assert run(product, [buf] * i + [0] + [buf] * (5 - i)) == 6, i
        assert run(product, [buf] * 5 + [buf + 4]) == 1
        small = M.MatmulBlocks(M.bf16, 4, 40, 128)
        assert small.workspace_bytes() == 0
        cast_op = M.CastBlocks(M.f32, 4, 40)
        for i in range(3):
            assert run(cast_op, [buf] * i + [0] + [buf] * (2 - i)) == 6, i
        assert M.launch_count() == before
        with pytest.raises(M.MorelloError) as err:
            op.run_async(full[:12] + [buf + 8])
        assert err.value.status == 1 and "16-byte" in str(err.value)
    assert lib.mrl_experts_check(None) == 6


@pytest.mark.parametrize("make", [
    lambda: M.CastBlocks(M.bf16, 300, 700), lambda: M.CastBlocks(M.f32, 300, 700, block_rows=128), lambda: M.MatmulBlocks(M.bf16, 8, 500, 384), lambda: M.MatmulBlocks(M.f32, 8, 500, 383),
    lambda: M.MatmulBlocks(M.bf16, 300, 500, 383), lambda: M.MatmulBlocks(M.f32, 300, 500, 384), lambda: M.MatmulBlocks(M.bf16, 4096, 4096, 256)])
def test_a_run_launches_what_its_plan_says(gpu, make):
    op = make()
    c = op._c
    sizes = [c.rows * c.cols * 4, c.rows * c.cols, c.rows * c.cols] if isinstance(op, M.CastBlocks) else [
        c.m * c.k, c.m * (c.k // 128 + 1) * 4, c.n * c.k, (c.n // 128 + 1) * (c.k // 128 + 1) * 4, c.m * c.n * 4, max(16, op.workspace_bytes())]
    with Device() as d:
        pointers = [d.put(np.zeros(n + 16, np.uint8)) for n in sizes]
        before = M.launch_count()
        op.run_device(pointers)
        assert M.launch_count() - before == len(op.plan().steps)
