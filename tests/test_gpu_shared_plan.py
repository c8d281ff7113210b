"""Attention over shared pages: how the work is dealt out.  Blocks with a piece of the shared keys and blocks without one take
unlike pieces of the requests' own keys, and pieces of shared keys have one, two, four or more steps: sizes on either side of
each choice, by the formula in 64 bits; calls beside one another."""
import pytest
import torch

from test_gpu_shared_attention import Problem, answers

pytestmark = pytest.mark.gpu


def apart(count, own):
    return [((), own + 3 * i, 1) for i in range(count)]


TREES = {
    # the few own keys find room where no shared ones are
    "short answers": answers(40, 60, lambda i: 1 + i % 20),
    # ... and do not: the blocks without shared keys take them all
    "answers as long as a quarter": answers(40, 30, lambda i: 90 + 5 * i),
    # ... or the others some as well
    "answers as long as the prompt": answers(48, 40, lambda i: 300 + 20 * i),
    "requests apart": answers(20, 30, lambda i: 40 + i) + apart(30, 400),
    # shared keys on every block, for many steps
    "a long prompt": answers(70, 260, lambda i: 30 + i),
    "two long prompts": [((("a", 200),), 25 * i + 1, 1) for i in range(9)] + [((("b", 90),), 400 + i, 1) for i in range(30)],
    # as many runs as an engine hands over in a step
    "many requests": answers(600, 3, lambda i: 1 + i % 7),
    "many pairs": [((("p%d" % (i // 2), 3),), 1 + i % 5, 1) for i in range(256)],
}


@pytest.mark.parametrize("heads,kv,dim,page,dtype", [(14, 2, 128, 16, "bf16"), (12, 2, 64, 8, "bf16"), (8, 1, 128, 64, "bf16"),
                                                     (6, 2, 64, 24, "bf16"), (6, 2, 48, 16, "bf16"), (6, 2, 64, 16, "f32"),
                                                     (20, 1, 64, 16, "bf16"), (3, 3, 64, 16, "bf16")])
@pytest.mark.parametrize("tree", list(TREES))
def test_against_the_formula(tree, heads, kv, dim, page, dtype):
    p = Problem(TREES[tree], heads, kv, dim, page, dtype, seed=len(tree) + heads)
    p.run()
    p.check()
    first = p.out.clone()
    p.out.fill_(5)
    assert torch.equal(p.run(early=True), first)


def test_calls_beside_one_another():
    """Two streams with a room each, call after call; then both in one graph."""
    problems = [Problem(TREES["answers as long as the prompt"], 14, 2, 128, 16, "bf16", seed=1),
                Problem(TREES["requests apart"], 12, 2, 64, 16, "bf16", seed=2)]
    alone = [p.run().clone() for p in problems]
    rooms = [p.room() for p in problems]
    tables = [torch.tensor(p.tables, device="cuda") for p in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    for p in problems:
        p.out.fill_(7)
    torch.cuda.synchronize()
    for turn in range(20):
        for p, room, table, stream in zip(problems, rooms, tables, streams):
            with torch.cuda.stream(stream):
                p.run(tables=table, room=room, early=bool(turn % 2))
    torch.cuda.synchronize()
    for p, want in zip(problems, alone):
        assert torch.equal(p.out, want) and not p.error.item()
        p.out.fill_(7)
    graph, main = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=main):
        streams[0].wait_stream(main)
        for turn in range(3):
            problems[1].run(tables=tables[1], room=rooms[1], early=True)
            with torch.cuda.stream(streams[0]):
                problems[0].run(tables=tables[0], room=rooms[0], early=True)
        main.wait_stream(streams[0])
    graph.replay()
    torch.cuda.synchronize()
    for p, want in zip(problems, alone):
        assert torch.equal(p.out, want) and not p.error.item()


@pytest.mark.parametrize("heads,kv,dim,page,dtype", [(14, 2, 128, 16, "bf16"), (12, 2, 64, 8, "bf16"), (8, 1, 128, 64, "bf16"), (28, 4, 128, 128, "bf16"),
                                                     (6, 2, 64, 24, "bf16"), (6, 2, 48, 4, "bf16"), (6, 2, 64, 16, "f32"), (40, 1, 64, 16, "bf16")])
@pytest.mark.parametrize("count", [2, 9, 60])
@pytest.mark.parametrize("cuts", [(1,), (5, 77, 130), (15, 16, 17, 18), (127, 128, 129, 255, 256), (300,)])
def test_runs_that_begin_and_end_anywhere(cuts, count, heads, kv, dim, page, dtype):
    """Shared keys in several runs around one another, cut inside of pages, tiles and steps; own keys from inside a page on."""
    p = Problem(answers(count, 512 // page + 1, lambda i: 1 + 7 * i), heads, kv, dim, page, dtype, seed=sum(cuts))
    runs, begin = [], 0
    for end in cuts:
        runs.append([0, count, begin, end, count - 1, len(runs) - 1])
        begin = end
    runs += [[i, 1, begin, n, i, len(cuts) - 1] for i, n in enumerate(p.lengths)]
    room = torch.empty(ops_module().shared_attention_room(count, len(runs), len(cuts), heads, kv, dim, p.dtype, shared=len(cuts)),
                       dtype=torch.uint8, device="cuda").fill_(255)
    p.run([torch.arange(count, dtype=torch.int32, device="cuda"), torch.tensor(runs, dtype=torch.int32, device="cuda"),
           torch.arange(len(cuts), len(cuts) + count, dtype=torch.int32, device="cuda")], room=room)
    p.check()


def ops_module():
    from from_scratch_inference_engine_b200.kernels import ops
    return ops
