"""Attention over pages that several requests share, against the formula in 64 bits."""
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from from_scratch_inference_engine_b200.cache.shared_runs import find_shared_runs

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def ops():
    from from_scratch_inference_engine_b200.kernels import ops as module
    return module


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


class Problem:
    """Requests whose pages are `tree`: a list of (path, own tokens, new tokens), a path being a tuple of (name, pages)."""

    def __init__(self, tree, heads, kv, dim, page, dtype, seed=0, entries=1, entry=0, least=1, std=1.0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.dim, self.page, self.dtype = heads, kv, dim, page, DTYPES[dtype]
        named, needed = {}, 0
        for path, own, new in tree:
            for name, pages in path:
                if name not in named:
                    named[name], needed = pages, needed + pages
            needed += -(-own // page)
        free = torch.randperm(needed + 2, generator=g).tolist()
        named = {name: [free.pop() for _ in range(pages)] for name, pages in named.items()}
        self.spare = free
        tables = []
        for path, own, new in tree:
            table = [p for name, _ in path for p in named[name]]
            tables.append(table + [free.pop() for _ in range(-(-own // page))])
        width = max(len(t) for t in tables) + 1
        self.tables = np.full((len(tree), width), -1, dtype=np.int32)
        for i, t in enumerate(tables):
            self.tables[i, :len(t)] = t
        self.new = [new for _, _, new in tree]
        self.lengths = [sum(pages for _, pages in path) * page + own for path, own, _ in tree]
        self.start = np.cumsum([0] + self.new[:-1]).astype(np.int32)
        self.pos0 = np.asarray([n - k for n, k in zip(self.lengths, self.new)], dtype=np.int32)
        self.positions = ints([p + t for p, n in zip(self.pos0, self.new) for t in range(n)])
        self.tokens = sum(self.new)
        self.found = find_shared_runs(self.tables, page, self.start, np.asarray(self.new), self.pos0, least)
        self.pages = (torch.randn(needed + 2, entries, 2, kv, page, dim, generator=g) * std).to(self.dtype).cuda()
        self.k, self.v = self.pages[:, entry, 0], self.pages[:, entry, 1]
        self.qkv = torch.randn(self.tokens, (heads + 2 * kv) * dim, generator=g).to(self.dtype).cuda()
        self.out = torch.full((self.tokens, heads * dim), 9.0, dtype=self.dtype, device="cuda")
        self.error = ints([0])
        self.lists = [ints(self.found.order), ints(self.found.runs).view(-1, 6), ints(self.found.own_run)]
        self.scale = dim ** -0.5

    def room(self, extra=0):
        f = self.found
        size = ops().shared_attention_room(len(f.order), len(f.runs), f.levels, self.heads, self.kv, self.dim, self.dtype)
        return torch.empty(size + extra, dtype=torch.uint8, device="cuda").fill_(255)

    def run(self, lists=None, tables=None, room=None, **options):
        order, runs, own_run = lists or self.lists
        return ops().shared_attention(self.qkv, self.qkv.stride(0), self.k, self.v, self.pages.stride(0), self.page,
                                      ints(self.tables) if tables is None else tables, self.positions, order, runs, own_run,
                                      self.out, self.heads, self.kv, self.dim, self.scale, self.room() if room is None else room,
                                      self.error, **options)

    def expected(self):
        """The formula, and how far the kernels' arithmetic may be off: weights rounded to bfloat16 (2^-8 of each) and the
        result rounded to the storage type; beside that 32-bit sums and exponentials.  Tensor cores may truncate: a whole
        step, 2^-23, for every addition."""
        group, step = self.heads // self.kv, 2.0 ** -23
        want = torch.zeros(self.tokens, self.heads * self.dim, dtype=torch.float64)
        bound = torch.zeros_like(want)
        k, v = self.k.double().cpu(), self.v.double().cpu()
        q = self.qkv[:, :self.heads * self.dim].double().cpu().view(self.tokens, self.kv, group, self.dim)
        for i, table in enumerate(self.tables.tolist()):
            held = [p for p in table if p >= 0]
            ki, vi = (x[held].permute(1, 0, 2, 3).reshape(self.kv, -1, self.dim) for x in (k, v))
            for t in range(self.start[i], self.start[i] + self.new[i]):
                n = int(self.positions[t]) + 1
                s = torch.einsum("kgd,knd->kgn", q[t], ki[:, :n]) * self.scale
                p = torch.softmax(s, -1)
                o = torch.einsum("kgn,knd->kgd", p, vi[:, :n])
                size = torch.einsum("kgn,knd->kgd", p, vi[:, :n].abs())
                # a score: dim products and additions; the exponents' arguments; twice, for numerator and denominator
                off = torch.einsum("kgd,knd->kgn", q[t].abs(), ki[:, :n].abs()).amax(-1, keepdim=True) * self.scale
                slack = 2 * (self.dim + 4) * step * off + 2 * (n + 64) * step + 2.0 ** -19
                unit = torch.finfo(self.dtype).eps / 2
                b = slack * size + unit * o.abs() * 1.01
                if self.dtype is torch.bfloat16:
                    b = b + 2.0 ** -8 * 1.01 * size
                want[t], bound[t] = o.reshape(-1), b.reshape(-1)
        return want, bound

    def check(self, want_bound=None):
        want, bound = want_bound or self.expected()
        got = self.out.double().cpu()
        assert int(self.error) == 0
        assert torch.isfinite(got).all()
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


def answers(count, prompt_pages, own, new=1):
    return [((("prompt", prompt_pages),), max(new, own(i)), new) for i in range(count)]


TREES = {
    "one token, nothing shared": [((), 1, 1)],
    "alone": [((), 70, 1), ((), 300, 1), ((), 5, 1)],
    "two of a page": answers(2, 1, lambda i: 1),
    "prompt": answers(5, 13, lambda i: 1 + 17 * i),
    "many rows": answers(37, 9, lambda i: 1 + i),
    "long": answers(3, 200, lambda i: 40 * i),
    "portions": answers(4, 6, lambda i: 3 + i, new=3),
    "tree": [((("s", 4), ("a", 7)), 3 + 9 * i, 1) for i in range(6)] + [((("s", 4), ("b", 2)), 60 - i, 1) for i in range(9)]
            + [((("s", 4),), 100 + i, 1) for i in range(3)] + [((), 33, 1), ((), 1, 1)],
    "deep": [(tuple((f"p{j}", 3) for j in range(i + 1)), 2 + i, 1 + i % 2) for i in range(8)],
    "own longer": answers(6, 2, lambda i: 500 + 60 * i),
}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,page", [(28, 4, 128, 16), (12, 2, 64, 8), (5, 5, 16, 4), (40, 1, 48, 16), (6, 2, 256, 1),
                                               (16, 1, 128, 64)])
@pytest.mark.parametrize("tree", list(TREES))
def test_against_the_formula(tree, heads, kv, dim, page, dtype):
    p = Problem(TREES[tree], heads, kv, dim, page, dtype, seed=len(tree) + dim)
    out = p.run()
    assert out is p.out
    p.check()


def test_the_same_every_time_and_whatever_the_room_held():
    p = Problem(TREES["tree"], 28, 4, 128, 16, "bf16")
    first = p.run().clone()
    for fill in (0, 127):
        room = p.room()
        room.fill_(fill)
        p.out.fill_(3)
        assert torch.equal(p.run(room=room), first)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores(dtype):
    """Scores far apart: weights that vanish, and maxima that move from piece to piece."""
    p = Problem(TREES["long"], 14, 2, 128, 16, dtype, seed=3, std=9.0)
    p.run()
    p.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_what_is_behind_the_last_key_is_not_read(dtype):
    """NaN in the rest of every last page, in pages that no request holds, in the other entry of a page."""
    p = Problem(TREES["portions"] + [((), 21, 1)], 12, 2, 64, 16, dtype, entries=2, entry=1)
    want = p.expected()
    p.pages[:, 0] = math.nan
    for page in p.spare:
        p.pages[page] = math.nan
    for table, n in zip(p.tables.tolist(), p.lengths):
        if n % 16:
            p.pages[table[n // 16], 1, :, :, n % 16:] = math.nan
    p.run()
    p.check(want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_token_does_not_see_what_the_token_behind_it_holds(dtype, bad):
    p = Problem([((("a", 2),), 5, 3), ((("a", 2),), 9, 1)], 12, 2, 64, 16, dtype)
    want, bound = p.expected()
    page, slot = p.tables[0, 2], 4                      # the last key of request 0
    p.v[page, :, slot] = bad
    p.k[page, :, slot] = bad
    p.run()
    got = p.out.double().cpu()
    ok = [0, 1, 3]
    assert ((got - want).abs() <= bound)[ok].all() and not torch.isfinite(got[2]).any()


def test_rows_of_tokens_that_are_not_listed_stay():
    p = Problem(TREES["prompt"], 12, 2, 64, 16, "bf16")
    order, runs, own_run = (x.clone() for x in p.lists)
    want = p.expected()
    wide = torch.full((9, 12 * 64 + 8), 5.0, dtype=torch.bfloat16, device="cuda")
    p.out = wide[2:7, :12 * 64]
    # the last request is not worked on: the places in front of it only
    first = p.found.runs[0].tolist()
    shorter = p.found.runs.copy()
    shorter[0, 1] -= 1
    keep = [r for r in range(len(shorter)) if r < p.found.shared or shorter[r, 0] < first[1] - 1]
    p.run([order[:-1].clone(), ints(shorter[keep]), own_run[:-1].clone()])
    left = int(order[-1])
    assert (wide[2 + left] == 5).all() and (wide[:2] == 5).all() and (wide[7:] == 5).all() and (wide[:, 12 * 64:] == 5).all()
    others = [t for t in range(5) if t != left]
    assert ((p.out.double().cpu() - want[0]).abs() <= want[1])[others].all()


def test_empty_runs_and_tokens_without_keys():
    """Runs without keys or places are passed over; a token that has no key gets zeros; runs may pad a list."""
    p = Problem(TREES["prompt"], 12, 2, 64, 16, "bf16")
    want = p.expected()
    order, runs, own_run = p.lists
    runs = torch.cat([runs, ints([[0, 0, 0, 0, 0, -1], [0, 1, 7, 7, 0, -1], [0, 1, 9, 3, 0, -1], [-5, 0, -5, 0, -5, -1]])])
    room = p.room(extra=1 << 22)
    p.run([order, runs, own_run], room=room)
    p.check(want)
    p.out.fill_(9)
    p.run([order, runs[-4:].clone(), torch.full_like(own_run, 1)])
    assert int(p.error) == 0 and (p.out == 0).all()
    p.out.fill_(9)
    p.run([order, runs[:0].clone(), torch.full_like(own_run, -1)])
    assert int(p.error) == 0 and (p.out == 0).all()
    p.run([order[:0].clone(), runs, own_run[:0].clone()], room=room)
    assert (p.out == 0).all()


def test_lists_that_point_outside():
    """What the lists get wrong is reported, and the rows that it does not concern are right."""
    p = Problem(TREES["prompt"] + [((), 50, 1)], 12, 2, 64, 16, "bf16")
    want, bound = p.expected()
    order, runs, own_run = p.lists
    alone = int(order.tolist().index(5))
    run = int(own_run[alone])
    for column, value in ((0, -1), (0, 7), (0, 2 ** 31 - 1), (1, 9), (1, 2 ** 31 - 1), (2, -1), (3, 10 ** 6), (3, 2 ** 31 - 1),
                          (4, 6), (4, -1), (5, run), (5, 10 ** 6), (5, -2)):
        broken = runs.clone()
        broken[run, column] = value
        p.error.zero_()
        p.out.fill_(9)
        p.run([order, broken, own_run])
        assert int(p.error) == 7, (column, value)
        assert ((p.out.double().cpu() - want).abs() <= bound)[:5].all()
    for value in (-1, 6, 2 ** 31 - 1):
        broken = order.clone()
        broken[alone] = value
        p.error.zero_()
        p.out.fill_(9)
        p.run([broken, runs, own_run])
        assert int(p.error) == 7 and (p.out[5] == 9).all()
        assert ((p.out.double().cpu() - want).abs() <= bound)[:5].all()
    for value in (len(runs), -1, -2 ** 31):                              # no such run: a token without keys
        broken = own_run.clone()
        broken[alone] = value
        p.error.zero_()
        p.run([order, runs, broken])
        assert ((p.out.double().cpu() - want).abs() <= bound)[:5].all()
    # a shared run that reaches to one of its tokens
    p.error.zero_()
    broken = runs.clone()
    broken[0, 3] += 16
    p.run([order, broken, own_run])
    assert int(p.error) == 7


def test_pages_outside_the_pool():
    p = Problem(TREES["prompt"], 12, 2, 64, 16, "f32")
    for value in (-1, len(p.pages), 2 ** 31 - 1, -2 ** 31):
        tables = ints(p.tables)
        tables[:, 3] = value                                             # keys 48 to 63 of the shared prompt
        p.error.zero_()
        p.run(tables=tables)
        assert int(p.error) == 3
        got = p.out.double().cpu()
        cut = p.k.clone()
        # the same without those keys
        k, v = (x.double().cpu() for x in (p.k, p.v))
        q = p.qkv[:, :12 * 64].double().cpu().view(5, 2, 6, 64)
        for i, table in enumerate(p.tables.tolist()):
            held = [pg for j, pg in enumerate(table) if pg >= 0 and j != 3]
            ki, vi = (x[held].permute(1, 0, 2, 3).reshape(2, -1, 64)[:, :p.lengths[i] - 16] for x in (k, v))
            o = torch.einsum("kgn,knd->kgd", torch.softmax(torch.einsum("kgd,knd->kgn", q[i], ki) * p.scale, -1), vi)
            assert (got[i] - o.reshape(-1)).abs().max() < 1e-5
        assert torch.equal(cut, p.k)


def test_room_for_fewer_levels_than_there_are():
    p = Problem([((("a", 2), ("b", 2), ("c", 2), ("d", 2)), 3, 1) for _ in range(2000)], 14, 2, 64, 16, "bf16")
    n = 2000
    # one run in another, all of all tokens
    runs = [[0, n, 32 * j, 32 * j + 32, 0, j - 1] for j in range(4)] + [[i, 1, 128, 131, i, 3] for i in range(100)]
    small = torch.empty(ops().shared_attention_room(n, len(runs), 0, 14, 2, 64, torch.bfloat16), dtype=torch.uint8, device="cuda")
    own = [4 + min(i, 99) for i in range(n)]
    p.run([ints(range(n)), ints(runs), ints(own)], room=small)
    assert int(p.error) == 8


def test_offsets_beyond_32_bits():
    """The last pages of a pool of more than 2^31 elements."""
    o = ops()
    pages = torch.empty(70000, 2, 4, 16, 256, dtype=torch.bfloat16, device="cuda")
    p = Problem(answers(3, 4, lambda i: 5 + i), 8, 4, 256, 16, "bf16")
    shift = 70000 - len(p.pages)
    pages[shift:] = p.pages[:, 0]
    tables = ints(np.where(p.tables >= 0, p.tables + shift, -1))
    o.shared_attention(p.qkv, p.qkv.stride(0), pages[:, 0], pages[:, 1], pages.stride(0), 16, tables, p.positions, *p.lists, p.out,
                       8, 4, 256, p.scale, p.room(), p.error)
    p.check()


def test_replayed_with_other_lists_and_on_another_stream():
    """A captured call goes by what the lists hold when it is replayed; two graphs have a room each."""
    p = Problem(TREES["tree"], 12, 2, 64, 16, "bf16")
    other = Problem(TREES["tree"], 12, 2, 64, 16, "bf16", seed=9, least=200)
    other.pages.copy_(p.pages)
    rows = max(len(p.found.runs), len(other.found.runs))
    order, own_run = p.lists[0].clone(), p.lists[2].clone()
    runs, tables = torch.zeros(rows, 6, dtype=torch.int32, device="cuda"), ints(p.tables)
    size = ops().shared_attention_room(len(order), rows, max(p.found.levels, other.found.levels), 12, 2, 64, torch.bfloat16)
    rooms = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    graphs = []
    side = torch.cuda.Stream()
    for room in rooms:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            p.run([order, runs, own_run], tables, room)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p.run([order, runs, own_run], tables, room, early=True)
        graphs.append(graph)
    queries = [p.qkv.clone(), other.qkv]
    for turn in range(4):
        held = other if turn % 2 else p
        runs.zero_()
        runs[:len(held.found.runs)] = held.lists[1]
        order.copy_(held.lists[0])
        own_run.copy_(held.lists[2])
        tables.copy_(ints(held.tables))
        p.qkv.copy_(queries[turn % 2])
        p.out.fill_(9)
        graphs[turn // 2].replay()
        p.check(held.expected())


def test_refusals():
    o = ops()
    p = Problem(TREES["prompt"], 12, 2, 64, 16, "bf16")
    room, tables = p.room(), ints(p.tables)
    good = dict(q=p.qkv, q_ld=p.qkv.stride(0), k_pages=p.k, v_pages=p.v, page_stride=p.pages.stride(0), page_size=16,
                block_tables=tables, positions=p.positions, order=p.lists[0], runs=p.lists[1], own_run=p.lists[2], out=p.out,
                heads=12, kv_heads=2, head_dim=64, scale=p.scale, room=room, error=p.error)
    o.shared_attention(**good)
    before = p.out.clone()
    bad = [dict(q=p.qkv.float()), dict(q=p.qkv.half(), k_pages=p.k.half(), v_pages=p.v.half(), out=p.out.half()), dict(q_ld=7),
           dict(q=p.qkv.cpu()), dict(k_pages=p.k.float()), dict(v_pages=p.v[:-1]), dict(page_size=8), dict(page_stride=1),
           dict(k_pages=p.k.transpose(2, 3)), dict(block_tables=tables.long()), dict(block_tables=tables[0]),
           dict(positions=p.positions[None]), dict(order=p.lists[0][:-1]), dict(runs=p.lists[1].view(-1)), dict(runs=p.lists[1].cpu()),
           dict(runs=torch.zeros(1025, 6, dtype=torch.int32, device="cuda")), dict(own_run=p.lists[2].float()), dict(out=p.out[:-1]),
           dict(out=p.out[:, :-8]), dict(heads=13), dict(kv_heads=0), dict(head_dim=24), dict(head_dim=272), dict(scale=0.0),
           dict(scale=-1.0), dict(scale=math.nan), dict(room=room[:100]), dict(room=room.float()), dict(room=room[1:].clone()[1:]),
           dict(error=p.error.long())]
    for change in bad:
        with pytest.raises(o.KernelError):
            o.shared_attention(**{**good, **change})
    # rows that start on no 16 bytes
    wide = torch.zeros(5, p.qkv.shape[1] + 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(o.KernelError):
        o.shared_attention(**{**good, "q": wide[:, 1:], "q_ld": wide.stride(0)})
    assert torch.equal(p.out, before) and int(p.error) == 0
    for args in ((-1, 1, 1, 12, 2, 64, torch.bfloat16), (1, 1025, 1, 12, 2, 64, torch.bfloat16), (1, 1, 1, 13, 2, 64, torch.bfloat16),
                 (1, 1, 1, 12, 2, 64, torch.float16), (1, 1, -1, 12, 2, 64, torch.float32)):
        with pytest.raises(o.KernelError):
            o.shared_attention_room(*args)


def formula_without(p, tables):
    """`Problem.expected` over the keys whose pages `tables` has inside the pool; zeros where none is left."""
    group, step, unit = p.heads // p.kv, 2.0 ** -23, torch.finfo(p.dtype).eps / 2
    want = torch.zeros(p.tokens, p.heads * p.dim, dtype=torch.float64)
    bound = torch.zeros_like(want)
    k, v = p.k.double().cpu(), p.v.double().cpu()
    q = p.qkv[:, :p.heads * p.dim].double().cpu().view(p.tokens, p.kv, group, p.dim)
    for i, table in enumerate(tables.tolist()):
        for t in range(p.start[i], p.start[i] + p.new[i]):
            keys = [(table[j // p.page], j % p.page) for j in range(int(p.positions[t]) + 1) if 0 <= table[j // p.page] < len(p.pages)]
            if not keys:
                continue
            pages, places = (torch.tensor(x) for x in zip(*keys))
            ki, vi = (x[pages, :, places].transpose(0, 1) for x in (k, v))
            weights = torch.softmax(torch.einsum("kgd,knd->kgn", q[t], ki) * p.scale, -1)
            o, size = torch.einsum("kgn,knd->kgd", weights, vi), torch.einsum("kgn,knd->kgd", weights, vi.abs())
            off = torch.einsum("kgd,knd->kgn", q[t].abs(), ki.abs()).amax(-1, keepdim=True) * p.scale
            b = (2 * (p.dim + 4) * step * off + 2 * (len(keys) + 64) * step + 2.0 ** -19) * size + unit * o.abs() * 1.01
            want[t], bound[t] = o.reshape(-1), (b + (2.0 ** -8 * 1.01 * size if p.dtype is torch.bfloat16 else 0)).reshape(-1)
    return want, bound


@pytest.mark.parametrize("dtype,heads,kv,dim,page", [("bf16", 28, 4, 128, 16), ("bf16", 28, 4, 64, 8), ("bf16", 14, 2, 128, 64), ("bf16", 14, 2, 128, 24),
                                                     ("bf16", 8, 2, 256, 16), ("f32", 14, 2, 128, 16), ("f32", 6, 2, 48, 8)])
@pytest.mark.parametrize("tree", ["many rows", "long", "tree"])
def test_keys_of_pages_outside_the_pool_are_left_out(tree, dtype, heads, kv, dim, page):
    """In every form alike, of shared runs and of a request's own keys: a page here and there, all shared ones, all."""
    p = Problem(TREES[tree], heads, kv, dim, page, dtype, seed=dim + page)
    held = p.tables >= 0
    shared = np.zeros_like(held)
    for first, count, begin, end, row, _ in p.found.runs[:p.found.shared]:
        pages = p.tables[row, begin // page:end // page]
        shared |= np.isin(p.tables, pages)
    for turn, gone in enumerate((held & (p.tables % 5 == 2), shared & held, held)):
        tables = p.tables.copy()
        tables[gone] = np.resize([-1, len(p.pages), 2 ** 31 - 1, -2 ** 31], gone.sum())
        p.error.zero_()
        p.out.fill_(9)
        p.run(tables=ints(tables))
        assert int(p.error) == 3
        want, bound = formula_without(p, tables)
        got = p.out.double().cpu()
        assert bool(((got - want).abs() <= bound).all()), (turn, float((got - want).abs().max()))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_runs_that_a_token_is_not_in(dtype):
    """An innermost run that there is none of, or one of another token, and a run around it that lies elsewhere are reported;
    -1 and runs without places are not."""
    p = Problem(TREES["tree"], 12, 2, 64, 16, dtype)
    want, bound = p.expected()
    order, runs, own_run = p.lists
    place = order.tolist().index(18)                                     # the request of 33 tokens that shares nothing
    run, elsewhere = int(own_run[place]), p.found.shared - 1
    assert runs[run].tolist()[1] == 1 and runs[run].tolist()[5] == -1
    first, count = runs[elsewhere].tolist()[:2]
    assert count > 1 and not first <= place < first + count
    others = [t for t in range(p.tokens) if t != 18]

    def reports(code, lists):
        p.error.zero_()
        p.out.fill_(9)
        p.run(lists)
        assert int(p.error) == code
        assert ((p.out.double().cpu() - want).abs() <= bound)[others].all()
    for value in (len(runs), 2 ** 31 - 1, -2, -2 ** 31, int(own_run[(place + 1) % p.tokens]), elsewhere):
        broken = own_run.clone()
        broken[place] = value
        reports(7, [order, runs, broken])
    broken = runs.clone()
    broken[run, 5] = elsewhere
    reports(7, [order, broken, own_run])
    broken = own_run.clone()
    broken[place] = -1
    reports(0, [order, runs, broken])
    assert (p.out[18] == 0).all()
    emptied = runs.clone()
    emptied[run, 1] = 0
    reports(0, [order, emptied, own_run])
    assert (p.out[18] == 0).all()


FIRST_CALLS = """
import sys, threading
import torch
sys.path[:0] = sys.argv[1:]
import test_gpu_shared_attention as t
forms = [(16, "bf16"), (24, "bf16"), (16, "f32")]               # on tcgen05, on mma.sync, FFMA
problems = [t.Problem(t.TREES["tree"], 28, 4, 128, *forms[i % 3]) for i in range(12)]
tables = [t.ints(p.tables) for p in problems]
rooms = [torch.empty(64 << 20, dtype=torch.uint8, device="cuda") for _ in problems]
torch.cuda.synchronize()
sizes, raised, start = [0] * 12, [], threading.Barrier(12)

def call(i):
    p, f = problems[i], problems[i].found
    size = lambda: t.ops().shared_attention_room(len(f.order), len(f.runs), f.levels, 28, 4, 128, p.dtype)
    try:
        start.wait()
        if i < 6:
            sizes[i] = size()
        p.run(tables=tables[i], room=rooms[i])
        sizes[i] = sizes[i] or size()
    except Exception as e:
        raised.append(e)

threads = [threading.Thread(target=call, args=(i,)) for i in range(12)]
for thread in threads:
    thread.start()
for thread in threads:
    thread.join()
assert not raised, raised
assert max(sizes) <= 64 << 20 and all(sizes[i] == sizes[i % 3] for i in range(12)), sizes
for p in problems:
    p.check()
print("well")
"""


def test_first_calls_of_several_threads_at_once():
    """In a process of its own, where nothing is known yet of how the launches look."""
    here = Path(__file__).resolve().parent
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS, str(here), str(here.parent)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "well", done.stderr[-2000:]
