"""What a program does between steps over a cache in pages: tokens that went without one come again, recorded steps follow each other."""
import numpy as np
import pytest

import morello_amd as M
from paged_util import POISON
from test_gpu_graph_capture import hip_runtime
from test_gpu_paged_step import LAYERS, Program, Recorded, same

pytestmark = pytest.mark.gpu


def run_step(program, number, added):
    program.inputs(number, added)
    for layer in range(LAYERS):
        program.upload(f"out{layer}", np.full_like(program.host[f"out{layer}"], POISON[program.dtype]))
    program.enqueue(None)
    M.synchronize()
    assert program.check() == sum(added)


@pytest.mark.parametrize("page,pages,wanted", [(16, 4, [20, 20, 10]), (7, 3, [11, 11, 5])])
def test_tokens_without_a_page_come_again(gpu, page, pages, wanted):
    """Fewer pages than three prompts want: what has no slot is not counted as cached, and passed again when a request has ended.  (Counted, its columns would never be drawn.)"""
    program = Program("bf16", 3, 60, 4, 2, 64, page, pages, 5, seed=41)
    wanted = np.array(wanted)
    run_step(program, 0, wanted)
    starts, slots = program.read("starts"), program.read("slots")
    assert program.read("left")[1] > 0
    inside = np.array([(slots[a:b] >= 0).sum() for a, b in zip(starts, starts[1:])])
    assert all((slots[a:a + n] >= 0).all() for a, n in zip(starts, inside)) and (inside < wanted).any()
    # the first request ends, its pages go back on the list
    table = program.read("table")
    back = table[0][table[0] >= 0]
    program.upload("free", np.concatenate([back, np.zeros(pages - len(back), np.int32)]))
    program.upload("count", [len(back), 0])
    program.upload("cached", [0, inside[1], inside[2]])
    run_step(program, 1, [0, wanted[1] - inside[1], wanted[2] - inside[2]])
    table, slots, lengths = program.read("table"), program.read("slots"), program.read("lengths")
    assert program.read("left")[1] == 0 and (slots[:int(program.read("starts")[-1])] >= 0).all()
    for r in (1, 2):   # every key has a place of its own
        assert lengths[r] == wanted[r]
        assert (table[r, :-(-wanted[r] // page)] >= 0).all()
    assert len(set(table[1][table[1] >= 0]) | set(table[2][table[2] >= 0])) == sum(-(-wanted[1:] // page))
    program.free()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_recorded_steps_follow_each_other_without_the_host(gpu, dtype):
    """Two recordings whose lengths and free counts change places, launched in turn and not waited for: each step begins where the one before it ended."""
    hip = hip_runtime()
    make = lambda: Program(dtype, 5, 24, 4, 1, 64, 16, 60, 80, seed=42, max_new=16)
    recorded, eager = make(), make()
    for p in (recorded, eager):   # prompts first, so that there is something cached
        run_step(p, 0, [16, 1, 3, 0, 2])
        p.advance()
        p.inputs(1, [1, 1, 4, 3, 0])
        for layer in range(LAYERS):
            p.upload(f"out{layer}", np.full_like(p.host[f"out{layer}"], POISON[dtype]))
    def swap(p):
        b = p.buffers
        b["cached"], b["lengths"], b["count"], b["left"] = b["lengths"], b["cached"], b["left"], b["count"]

    stream = M.Stream()
    graphs = []
    for _ in range(2):
        graphs.append(Recorded(hip, recorded, stream))
        swap(recorded)
    steps = 9   # (an odd number: the last one's lengths are where the first recording puts them)
    for i in range(steps):
        graphs[i % 2].launch(stream)
    stream.synchronize()
    for i in range(steps):
        eager.enqueue(None)
        M.synchronize()
        assert eager.check() == 9
        if i + 1 < steps:
            eager.advance()
    assert same(recorded.results(), eager.results())
    assert eager.read("lengths").tolist() == [16 + steps, 1 + steps, 3 + 4 * steps, 3 * steps, 2]
    for g in graphs:
        g.destroy()
    recorded.free()
    eager.free()
    stream.destroy()
