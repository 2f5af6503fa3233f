"""Steps of a serving program: page tables, then rotary positions and attention in each of two layers, over prompts and single tokens;
eager, and recorded into graphs that are replayed while lengths change."""
import ctypes as C

import numpy as np
import pytest

import morello_amd as M
from paged_util import DTYPE, POISON, STORED, Batch, as_f64, values
from test_gpu_graph_capture import hip_runtime
from test_gpu_page_tables import by_hand
from test_gpu_rotary import bound as rotary_bound
from test_gpu_rotary import frequencies_of, turned

pytestmark = pytest.mark.gpu

LAYERS = 2


class Program:
    """The device buffers and operators of a program that serves `requests` requests, and what it knows of them on the host."""

    def __init__(self, dtype, requests, tokens, q_heads, kv_heads, dim, page, pages, width, seed, max_new=0, window=0):
        self.dtype, self.requests, self.tokens, self.page, self.pages, self.seed, self.window = dtype, requests, tokens, page, pages, seed, window
        self.q_heads, self.kv_heads, self.dim, self.width = q_heads, kv_heads, dim, width
        self.tables = M.PageTables(requests, width, page, pages, tokens, pages)
        self.rotary = M.Rotary(DTYPE[dtype], tokens, q_heads, kv_heads, dim, [dim // 4, dim // 8], page_size=page, pages=pages)
        self.attention = M.PagedAttention(DTYPE[dtype], tokens, requests, q_heads, kv_heads, dim, page, pages, width, max_new=max_new, window=window)
        free = np.random.default_rng(seed).permutation(pages).astype(np.int32)
        host = {"cached": np.zeros(requests, np.int32), "added": np.zeros(requests, np.int32), "free": free, "count": np.array([pages, 0], np.int32),
                "table": np.full((requests, width), -1, np.int32), "starts": np.zeros(requests + 1, np.int32), "lengths": np.zeros(requests, np.int32),
                "slots": np.zeros(tokens, np.int32), "positions": np.zeros((2, tokens), np.int32), "left": np.zeros(2, np.int32),
                "frequencies": frequencies_of(dim // 4 + dim // 8)}
        for layer in range(LAYERS):
            for name, heads in (("q", q_heads), ("k", kv_heads), ("v", kv_heads), ("turned", q_heads), ("out", q_heads)):
                host[f"{name}{layer}"] = np.full((tokens, heads, dim), POISON[dtype], STORED[dtype])
            for name in ("keys", "values"):
                host[f"{name}{layer}"] = np.full((pages, page, kv_heads, dim), POISON[dtype], STORED[dtype])
        host["workspace"] = np.full(max(16, self.attention.workspace_bytes()), 0xff, np.uint8)
        self.host, self.buffers = host, {name: M.DeviceBuffer.from_numpy(a) for name, a in host.items()}

    def upload(self, name, array):
        array = np.ascontiguousarray(array, self.host[name].dtype)
        assert array.shape == self.host[name].shape
        M._check(M.B.load().mrl_memcpy_h2d(self.buffers[name].ptr, array.ctypes.data, array.nbytes), "mrl_memcpy_h2d")
        self.host[name] = array

    def read(self, name):
        return self.buffers[name].to_numpy(self.host[name].dtype, self.host[name].shape)

    def inputs(self, step, added):
        """What the step's new tokens bring; positions on their second axis, any."""
        self.upload("added", added)
        rows = int(np.sum(added))
        second = np.random.default_rng([self.seed, step]).integers(0, 900, self.tokens)
        positions = self.read("positions")
        positions[1] = second
        self.upload("positions", positions)
        for layer in range(LAYERS):
            for i, name in enumerate("qkv"):
                x = values(self.dtype, self.seed + 10 * step + layer, i, self.host[f"{name}{layer}"].shape)[0]
                x[rows:] = POISON[self.dtype]
                self.upload(f"{name}{layer}", x)

    def enqueue(self, stream):
        p = {name: b.ptr for name, b in self.buffers.items()}
        self.tables.run_async([p[n] for n in ("cached", "added", "free", "count", "table", "starts", "lengths", "slots", "positions", "left")], stream)
        for layer in range(LAYERS):
            of = lambda *names: [p[f"{n}{layer}"] for n in names]
            self.rotary.run_async(of("q", "k", "v") + [p["positions"], p["frequencies"], p["slots"]] + of("turned", "keys", "values"), stream)
            self.attention.run_async(of("turned", "keys", "values") + [p["table"], p["starts"], p["lengths"]] + of("out") + [p["workspace"]], stream)

    def advance(self):
        self.upload("cached", self.read("lengths"))
        self.upload("count", [self.read("left")[0], 0])

    def results(self):
        return {name: self.read(name) for name in ["table", "starts", "lengths", "slots", "left"] + [f"{n}{i}" for i in range(LAYERS) for n in ("turned", "out", "keys", "values")]}

    def check(self):
        """Tables, rotary and attention of the step just run, each from what the one before left; -> rows."""
        h = self.host
        got = self.results()
        positions = self.read("positions")
        want = by_hand(self.tables, h["cached"], h["added"], h["free"], int(h["count"][0]), h["table"])
        for name, g, w in zip(("table", "starts", "lengths", "slots", "positions", "left"),
                              (got["table"], got["starts"], got["lengths"], got["slots"], positions[0], got["left"]), want):
            assert np.array_equal(g, w), name
        h["table"] = got["table"]
        rows = int(got["starts"][-1])
        sections = [self.dim // 4, self.dim // 8]
        for layer in range(LAYERS):
            keys, vals = (got[f"{n}{layer}"].reshape(-1, self.kv_heads, self.dim) for n in ("keys", "values"))
            before_k, before_v = (h[f"{n}{layer}"].reshape(-1, self.kv_heads, self.dim).copy() for n in ("keys", "values"))
            slots = got["slots"][:rows]
            new = slots[slots >= 0]
            for name, g in (("q", got[f"turned{layer}"][:rows]), ("k", keys[slots])):
                y, size = turned(as_f64(self.dtype, h[f"{name}{layer}"][:rows]), positions[:, :rows], h["frequencies"], sections, False)
                off = np.abs(as_f64(self.dtype, g) - y) <= rotary_bound(y, size, self.dtype)
                assert off[slots >= 0].all() if name == "k" else off.all(), (name, layer)
            before_k[new], before_v[new] = keys[new], h[f"v{layer}"][:rows][slots >= 0]
            assert np.array_equal(keys, before_k, equal_nan=self.dtype == "f32") and np.array_equal(vals, before_v, equal_nan=self.dtype == "f32")
            h[f"keys{layer}"], h[f"values{layer}"] = got[f"keys{layer}"], got[f"values{layer}"]
            b = Batch.__new__(Batch)
            b.dtype, b.tokens, b.q_heads, b.kv_heads, b.dim, b.page, b.pages, b.width = (
                self.dtype, self.tokens, self.q_heads, self.kv_heads, self.dim, self.page, self.pages, self.width)
            b.requests, b.heads_first, b.starts, b.totals, b.table = self.requests, False, got["starts"], got["lengths"], got["table"]
            b.keys, b.values, b.q64 = got[f"keys{layer}"], got[f"values{layer}"], as_f64(self.dtype, got[f"turned{layer}"])
            want_out, bound = b.want(self.window)
            g = as_f64(self.dtype, got[f"out{layer}"])
            assert (np.abs(g[:rows] - want_out[:rows]) <= bound[:rows]).all(), layer
            assert np.isnan(g[rows:]).all(), "rows behind the last token were written"
        return rows

    def free(self):
        for b in self.buffers.values():
            b.free()


STEPS = [   # new tokens of five requests: prompts, prompts beside single tokens, single tokens, none, a request that waits
    [40, 0, 17, 3, 1], [1, 70, 1, 1, 0], [1, 1, 1, 1, 30], [1, 1, 1, 1, 1], [0, 1, 0, 0, 1], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1]]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,window", [(4, 2, 64, 16, 0), (8, 1, 128, 16, 50), (3, 3, 40, 7, 0)])
def test_prompts_then_tokens(gpu, dtype, q_heads, kv_heads, dim, page, window):
    stream = M.Stream()
    program = Program(dtype, 5, 80, q_heads, kv_heads, dim, page, 40, 12, seed=31, window=window)
    for step, added in enumerate(STEPS):
        program.inputs(step, added)
        for layer in range(LAYERS):
            program.upload(f"out{layer}", np.full_like(program.host[f"out{layer}"], POISON[dtype]))
        program.enqueue(stream)
        stream.synchronize()
        assert program.check() == sum(added)
        program.advance()
    program.free()
    stream.destroy()


def test_a_cache_that_runs_out(gpu):
    """The last pages go to the first requests; tokens without one have no slot, and attend to the keys that there are."""
    program = Program("bf16", 3, 60, 2, 1, 64, 16, 4, 3, seed=32)
    for step, added in enumerate([[20, 20, 10], [30, 1, 1]]):
        program.inputs(step, added)
        for layer in range(LAYERS):
            program.upload(f"out{layer}", np.full_like(program.host[f"out{layer}"], POISON["bf16"]))
        program.enqueue(None)
        M.synchronize()
        program.check()
        assert program.read("left")[1] > 0
        program.advance()
    program.free()


class Recorded:
    def __init__(self, hip, program, stream):
        self.hip, self.graph, self.exec = hip, C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(stream.handle, 0) == 0   # hipStreamCaptureModeGlobal
        try:
            program.enqueue(stream)
        finally:
            assert hip.hipStreamEndCapture(stream.handle, C.byref(self.graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, 0) == 0

    def launch(self, stream):
        assert self.hip.hipGraphLaunch(self.exec, stream.handle) == 0

    def destroy(self):
        self.hip.hipGraphExecDestroy(self.exec)
        self.hip.hipGraphDestroy(self.graph)


def same(a, b):
    return all(np.array_equal(a[name].view(np.uint8), b[name].view(np.uint8)) for name in a)


@pytest.mark.parametrize("dtype,max_new", [("bf16", 0), ("bf16", 8), ("f32", 0)])
def test_graphs_replayed_while_lengths_change(gpu, dtype, max_new):
    """Two recorded programs side by side, each with a workspace of its own, and the same steps run eagerly between their replays."""
    hip = hip_runtime()
    steps = STEPS if max_new == 0 else [[8, 0, 5, 3, 1], [1, 7, 1, 1, 0], [1, 1, 1, 1, 8], [1, 1, 1, 1, 1], [0, 1, 0, 0, 1], [2, 1, 1, 1, 1]]
    make = lambda seed: Program(dtype, 5, 80, 4, 1, 64, 16, 200, 80, seed=seed, max_new=max_new)
    recorded, eager = [make(33), make(34)], [make(33), make(34)]
    assert recorded[0].attention.workspace_bytes() > 0
    streams = [M.Stream(), M.Stream()]
    graphs = [Recorded(hip, p, s) for p, s in zip(recorded, streams)]
    for step, added in enumerate(steps):
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
        for p in recorded + eager:
            p.advance()
    for g in graphs:
        g.destroy()
    for p in recorded + eager:
        p.free()
    for s in streams:
        s.destroy()


def test_a_step_run_again_gives_the_same(gpu):
    """Keys shared out over workgroups meet in a fixed order: a second run has the first one's bits, whatever the workspace held."""
    program = Program("bf16", 2, 8, 4, 1, 128, 16, 700, 650, seed=35, max_new=1)
    program.upload("table", np.stack([np.arange(650), np.full(650, 699)]))
    for layer in range(LAYERS):
        for i, name in enumerate(("keys", "values")):
            program.upload(f"{name}{layer}", values("bf16", 35, 5 + i + 2 * layer, program.host[f"{name}{layer}"].shape)[0])
    program.upload("cached", [10000, 3])
    program.inputs(0, [1, 1])
    assert "k_paged_attn_merge" in " ".join(program.attention.plan().kernels)
    program.enqueue(None)
    M.synchronize()
    first = program.results()
    for fill in (0x00, 0x7f):
        program.upload("workspace", np.full_like(program.host["workspace"], fill))
        program.enqueue(None)
        M.synchronize()
        again = program.results()
        assert same({n: first[n] for n in ("out0", "out1")}, {n: again[n] for n in ("out0", "out1")})
    program.free()
