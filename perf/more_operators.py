"""The operators of answers to one prompt, as cases that can be timed and checked.

Kinds of cases:

  shared   attention of new tokens over a paged cache in which requests hold the same leading pages: the keys and
           values that several requests share are read, and multiplied, once for all of them
  count    tokens counted into the requests' histories: how often each was generated, and whether it occurred at all
  adjust   logits changed in place by those histories (penalties for repeated tokens), by biases and by masks of the
           allowed tokens

Sizes are those of the 1.5B, 7B and 14B layer stacks and their vocabularies, and generic ones.  Everything is drawn from
the seed on the device.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False
DEVICE = "cuda:0"
F64 = torch.float64
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ROOM = 1 << 28              # bytes of working memory that a program of these sizes keeps


# ------------------------------------------------------------------------------------------ cases
def _shared(name, heads, kv, dim, page, common, branches, own_low, own_high, new, dtype):
    """`common` tokens that all requests share; `branches`: "tokens*requests" each, tokens that so many of them share
    behind those; own_low to own_high tokens of every request's own, the last `new` of which are this step's."""
    return {"name": name, "kind": "shared", "heads": heads, "kv": kv, "dim": dim, "page": page, "common": common,
            "branches": branches, "own_low": own_low, "own_high": own_high, "new": new, "dtype": dtype}


def listed():
    return [
        # two answers to a short prompt at the 7B layer's heads: latency
        _shared("pair_300", 28, 4, 128, 16, 0, "300*2", 1, 40, 1, "bf16"),
        # eight answers to a prompt of 4,096 tokens at the 7B layer's heads
        _shared("samples_8x4096", 28, 4, 128, 16, 0, "4096*8", 16, 400, 1, "bf16"),
        # sixty-four answers that have grown about as long as the prompt they share
        _shared("samples_64x2048", 28, 4, 128, 16, 0, "2048*64", 32, 2048, 1, "bf16"),
        # a full batch of one long document at the 14B layer's heads
        _shared("samples_200x8192", 40, 8, 128, 16, 0, "8192*200", 32, 512, 1, "bf16"),
        # a system prompt that all share, four prompts behind it with twelve answers each, at the 1.5B layer's heads
        _shared("tree_48", 12, 2, 128, 16, 512, "1500*12 700*12 64*12 0*12", 1, 600, 1, "bf16"),
        # the 32-bit path, an odd number of answers, small pages
        _shared("samples_f32_23", 12, 2, 128, 8, 0, "1000*23", 1, 200, 1, "f32"),
        # a decode step's 64 chosen tokens
        {"name": "count_step_64", "kind": "count", "tokens": 64, "slots": 64, "vocab": 152064, "generated": True},
        # forty prompts taken in
        {"name": "count_prompts", "kind": "count", "tokens": 32768, "slots": 40, "vocab": 151936, "generated": False},
        # one user's row
        _adjust("adjust_1", 1, 151936, 400, 0, 0, 0),
        # a batch of 64 with all there is: histories, biases, every third row under a grammar
        _adjust("adjust_64", 64, 152064, 1500, 40, 22, 20000),
        # every row under a grammar that allows few tokens
        _adjust("adjust_grammar_24", 24, 151936, 300, 0, 24, 90),
        # an odd vocabulary: rows that start on no 16 bytes
        _adjust("adjust_odd_33", 33, 32003, 700, 300, 11, 16000),
    ]


def _adjust(name, rows, vocab, distinct, biases, masked, allowed):
    """`distinct`: different tokens in a row's history; `biases`: per row; `masked`: rows with a mask, which leaves
    `allowed` tokens."""
    return {"name": name, "kind": "adjust", "rows": rows, "vocab": vocab, "distinct": distinct, "biases": biases,
            "masked": masked, "allowed": allowed}


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "count", "adjust", "adjust"])
    if kind == "count":
        case = {"kind": kind, "tokens": _log_int(rng, 1, 32768), "slots": _log_int(rng, 1, 64),
                "vocab": rng.choice([152064, 151936, 32003, 50001, _log_int(rng, 100, 150000)]), "generated": rng.random() < 0.6}
        return case
    if kind == "adjust":
        vocab = rng.choice([152064, 151936, 32003, 50001, _log_int(rng, 100, 150000)])
        rows = _log_int(rng, 1, 64)
        case = _adjust("", rows, vocab, _log_int(rng, 1, min(4000, vocab // 2)), rng.choice([0, 0, _log_int(rng, 1, 300)]),
                       rng.choice([0, rows, rng.randint(0, rows)]), _log_int(rng, 1, vocab))
        case["biases"] = min(case["biases"], vocab // 4)
        del case["name"]
        return case
    heads, kv = rng.choice([(28, 4), (28, 4), (12, 2), (40, 8), (8, 8), (16, 1), (6, 3)])
    dim, dtype = rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "bf16", "f32"])
    requests = _log_int(rng, 2, 128)
    most = 8192 * 64 * 28 // (requests * heads) // (8 if dtype == "f32" else 1)
    prefix = _log_int(rng, 20, max(40, min(8192, most)))
    form = rng.choice(["one", "one", "several", "tree", "alone"])
    common = 0
    if form == "one":
        branches = f"{prefix}*{requests}"
    elif form == "alone":                       # beside requests that share nothing
        apart = max(1, requests // 3)
        branches = " ".join([f"{prefix}*{requests - apart}"] + ["0*1"] * apart)
    else:
        parts = min(requests, rng.randint(2, 5))
        sizes = [requests // parts + (i < requests % parts) for i in range(parts)]
        branches = " ".join(f"{_log_int(rng, 8, prefix)}*{n}" for n in sizes)
        common = _log_int(rng, 8, prefix) if form == "tree" else 0
    new = rng.choice([1, 1, 1, 2])
    case = _shared("", heads, kv, dim, rng.choice([16, 16, 8, 32, 64]), common, branches, new,
                   new + _log_int(rng, 1, max(2, min(2000, most // 2))), new, dtype)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------- layouts
def _layout(case):
    """The requests of a `shared` case in the order of the tree, as (common pages, branch, branch pages, all tokens), and the
    pages of every branch's own.  Shared are full pages; what a prefix has beyond them every request holds itself."""
    page = case["page"]
    common = case["common"] // page
    requests, branch_pages, i = [], [], 0
    for b, text in enumerate(case["branches"].split()):
        tokens, count = (int(n) for n in text.split("*"))
        count_pages = (case["common"] + tokens) // page - common if count > 1 or tokens else 0
        branch_pages.append(count_pages)
        for _ in range(count):
            # own lengths spread evenly over the logarithm of their range, in no order
            part = math.modf(0.5 + i * 0.6180339887498949)[0]
            length = int(round(case["own_low"] * (case["own_high"] / case["own_low"]) ** part))
            requests.append((common, b, count_pages, case["common"] + tokens + max(case["new"], length)))
            i += 1
    return requests, branch_pages


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    error = _ints([0])
    if case["kind"] == "shared":
        return _prepare_shared(case, gen, error)
    vocab, words = case["vocab"], -(-case["vocab"] // 32)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=DEVICE)
    if case["kind"] == "count":
        n, slots = case["tokens"], case["slots"]
        # most tokens of a text are among the frequent ones
        tokens = (vocab * uniform(n) ** 3).to(torch.int32).clamp_(max=vocab - 1)
        of = torch.arange(n, device=DEVICE) * slots // n if n >= slots else torch.randperm(slots, generator=gen, device=DEVICE)[:n]
        return {"case": case, "tokens": tokens, "of": of.to(torch.int32), "error": error,
                "counts": torch.zeros(slots, vocab, dtype=torch.int32, device=DEVICE),
                "seen": torch.zeros(slots, words, dtype=torch.int32, device=DEVICE)}
    rows = case["rows"]
    order = uniform(rows, vocab)
    held = torch.zeros(rows, vocab, dtype=torch.bool, device=DEVICE)
    held.scatter_(1, order.topk(case["distinct"]).indices, True)
    # half of the history comes from the prompt and was not generated
    counts = (held & (uniform(rows, vocab) < 0.5)) * (1 + (4 * uniform(rows, vocab) ** 4).to(torch.int32))
    slots = torch.randperm(rows, generator=gen, device=DEVICE).to(torch.int32)
    state = {"case": case, "error": error, "slots": slots, "counts": counts.to(torch.int32), "seen": _packed(held),
             "logits": torch.empty(rows, vocab, device=DEVICE).normal_(0, 3, generator=gen),
             # penalties as requests name them, one row in four without
             "penalties": torch.stack([1 + 0.5 * uniform(rows), uniform(rows), 0.5 * uniform(rows)], 1)
             * (torch.arange(rows, device=DEVICE) % 4 != 3)[:, None], "bias": None, "masks": None}
    state["penalties"][:, 0].clamp_(min=1)
    if case["biases"]:
        tokens = uniform(rows, vocab).topk(case["biases"]).indices.sort(1).values.to(torch.int32)
        state["bias"] = (_ints([r * case["biases"] for r in range(rows + 1)]), tokens.reshape(-1).contiguous(),
                         torch.empty(tokens.numel(), device=DEVICE).normal_(0, 4, generator=gen))
    if case["masked"]:
        allowed = torch.zeros(case["masked"], vocab, dtype=torch.bool, device=DEVICE)
        allowed.scatter_(1, uniform(case["masked"], vocab).topk(case["allowed"]).indices, True)
        of = torch.full((rows,), -1, dtype=torch.int32, device=DEVICE)
        of[torch.randperm(rows, generator=gen, device=DEVICE)[:case["masked"]]] = _ints(list(range(case["masked"])))
        state["masks"] = (of, _packed(allowed))
    return state


def _packed(bits):
    """[rows, n] truth values as words of 32: bit v % 32 of word v // 32."""
    bits = F.pad(bits, (0, -bits.shape[1] % 32)).view(bits.shape[0], -1, 32)
    words = (bits.long() << torch.arange(32, device=DEVICE)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _unpacked(words, n):
    return ((words[:, :, None] >> torch.arange(32, device=DEVICE)) & 1).bool().flatten(1)[:, :n]


def _prepare_shared(case, gen, error):
    heads, kv, dim, page, new = (case[k] for k in ("heads", "kv", "dim", "page", "new"))
    requests, branch_pages = _layout(case)
    count = len(requests)
    # physical pages in no order: those all share, each branch's, each request's own
    needed = requests[0][0] + sum(branch_pages) + sum(-(-r[3] // page) - r[0] - r[2] for r in requests)
    pool = needed + 3
    free = torch.randperm(pool, generator=gen, device=DEVICE).tolist()
    common = [free.pop() for _ in range(requests[0][0])]
    branches = [[free.pop() for _ in range(n)] for n in branch_pages]
    place = torch.randperm(count, generator=gen, device=DEVICE).tolist()      # the tree's request i is the batch's place[i]
    width = max(-(-r[3] // page) for r in requests)
    tables, lengths = [None] * count, [0] * count
    for i, (_, b, _, length) in enumerate(requests):
        table = common + branches[b]
        table = table + [free.pop() for _ in range(-(-length // page) - len(table))]
        tables[place[i]], lengths[place[i]] = table + [-1] * (width - len(table)), length
    # who shares what: a run is `count` places of `order` from `first` on (tokens), the keys from `begin` to `end` that those
    # tokens see by it, the batch's row of the block tables to find them in, and the run around it
    runs, order, own_run = [], [], []
    sizes = [sum(r[1] == b for r in requests) for b in range(len(branch_pages))]
    root = -1
    if requests[0][0] and count > 1:
        runs.append([0, count * new, 0, common_end(case), place[0], -1])
        root = 0
    i = 0
    for b, size in enumerate(sizes):
        outer, begin = root, common_end(case) if root >= 0 else 0
        end = begin + branch_pages[b] * page
        if size > 1 and end > begin:
            runs.append([i * new, size * new, begin, end, place[i], outer])
            outer, begin = len(runs) - 1, end
        for _ in range(size):
            at, length = place[i], requests[i][3]
            runs.append([i * new, new, begin, length, at, outer])
            order += [at * new + t for t in range(new)]
            own_run += [len(runs) - 1] * new
            i += 1
    positions = [n - new + t for n in lengths for t in range(new)]
    dtype = DTYPES[case["dtype"]]
    qkv = torch.empty(count * new, (heads + 2 * kv) * dim, device=DEVICE).normal_(0, 1, generator=gen).to(dtype)
    pages = torch.empty(pool, 1, 2, kv, page, dim, dtype=dtype, device=DEVICE).normal_(0, 1, generator=gen)
    return {"case": case, "qkv": qkv, "pages": pages, "tables": _ints(tables), "positions": _ints(positions),
            "order": _ints(order), "runs": _ints(runs), "own_run": _ints(own_run), "error": error,
            "out": torch.empty(count * new, heads * dim, dtype=dtype, device=DEVICE),
            "room": torch.empty(ROOM, dtype=torch.uint8, device=DEVICE)}


def common_end(case):
    return case["common"] // case["page"] * case["page"]


# --------------------------------------------------------------------------------------- one pass
def run(s):
    return {"shared": _run_shared, "count": _run_count, "adjust": _run_adjust}[s["case"]["kind"]](s)


def _run_shared(s):
    c, pages = s["case"], s["pages"]
    heads, kv, dim, page, new = (c[k] for k in ("heads", "kv", "dim", "page", "new"))
    if own:
        from from_scratch_inference_engine_b200.kernels import ops
        return ops.shared_attention(s["qkv"], s["qkv"].stride(0), pages[:, 0, 0], pages[:, 0, 1], pages.stride(0), page,
                                    s["tables"], s["positions"], s["order"], s["runs"], s["own_run"], s["out"], heads, kv,
                                    dim, dim ** -0.5, s["room"], s["error"])
    tables = s["tables"]
    items, width = tables.shape
    at = tables.clamp(min=0).long()

    def rows(which):                              # [requests, kv, keys, dim]
        return pages[at, 0, which].permute(0, 2, 1, 3, 4).reshape(items, kv, width * page, dim).float()
    q = s["qkv"][:, :heads * dim].float().view(items, new, kv, heads // kv, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(items, kv, new * (heads // kv), dim)
    scores = (q @ rows(0).mT) * dim ** -0.5
    keys = torch.arange(width * page, device=DEVICE)
    unseen = keys > s["positions"].view(items, 1, new, 1, 1)
    scores = scores.view(items, kv, new, heads // kv, -1).masked_fill(unseen, -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    weights = (weights / weights.sum(-1, keepdim=True)).view(items, kv, new * (heads // kv), -1)
    out = (weights @ rows(1)).view(items, kv, new, heads // kv, dim).permute(0, 2, 1, 3, 4)
    return s["out"].copy_(out.reshape(items * new, heads * dim))


def _run_count(s):
    vocab = s["case"]["vocab"]
    if own:
        from from_scratch_inference_engine_b200.kernels import ops
        ops.count_tokens(s["tokens"], s["of"], s["counts"], s["seen"], s["error"], generated=s["case"]["generated"])
        return {"counts": s["counts"], "seen": s["seen"]}
    tokens, of = s["tokens"].long(), s["of"].long()
    if s["case"]["generated"]:
        s["counts"].index_put_((of, tokens), torch.ones_like(s["tokens"]), accumulate=True)
    held = _unpacked(s["seen"], vocab)
    held[of, tokens] = True
    s["seen"].copy_(_packed(held))
    return {"counts": s["counts"], "seen": s["seen"]}


def _run_adjust(s):
    logits = s["logits"]
    if own:
        from from_scratch_inference_engine_b200.kernels import ops
        return ops.adjust_logits(logits, s["error"], s["slots"], s["penalties"], s["counts"], s["seen"], s["bias"], s["masks"])
    rows, vocab = logits.shape
    slots = s["slots"].long()
    counts = s["counts"][slots]
    divisor, presence, frequency = s["penalties"][:, :, None].unbind(1)
    held = _unpacked(s["seen"][slots], vocab)
    repeated = torch.where(logits > 0, logits / divisor, logits * divisor) - presence * (counts > 0) - frequency * counts
    z = torch.where(held, repeated, logits)
    if s["bias"] is not None:
        start, tokens, values = s["bias"]
        row = torch.repeat_interleave(torch.arange(rows, device=DEVICE), s["case"]["biases"])
        z = z.index_put((row, tokens.long()), values, accumulate=True)
    if s["masks"] is not None:
        of, masks = s["masks"]
        allowed = _unpacked(masks, vocab)[of.clamp(min=0).long()] | (of < 0)[:, None]
        z = z.masked_fill(~allowed, -math.inf)
    return logits.copy_(z)


# ------------------------------------------------------------------------------- bytes, operations
def work(case):
    if case["kind"] == "count":
        # a token's id and slot; its word of the history, and its count, read and written
        return {"bytes": case["tokens"] * (8 + 8 + (8 if case["generated"] else 0)), "flops": case["tokens"]}
    if case["kind"] == "adjust":
        rows, vocab, words = case["rows"], case["vocab"], -(-case["vocab"] // 32)
        # every row's history and the masks; what occurred: its count, its logit read and written; biases: token, value and
        # a logit read and written; what a mask forbids is written
        moved = rows * (words * 4 + case["distinct"] * 12 + case["biases"] * 16) \
            + case["masked"] * (words * 4 + (vocab - case["allowed"]) * 4)
        return {"bytes": moved, "flops": rows * (5 * case["distinct"] + case["biases"])}
    requests, branch_pages = _layout(case)
    heads, kv, dim, page, new = (case[k] for k in ("heads", "kv", "dim", "page", "new"))
    size = DTYPES[case["dtype"]].itemsize
    keys = (requests[0][0] + sum(branch_pages)) * page + sum(r[3] - (r[0] + r[2]) * page for r in requests)
    seen = sum(r[3] - new + t + 1 for r in requests for t in range(new))
    return {"bytes": keys * kv * dim * 2 * size + 2 * len(requests) * new * heads * dim * size, "flops": 4 * seen * heads * dim}


# -------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "shared":
        return _exact_shared(case, s)
    vocab = case["vocab"]
    if case["kind"] == "count":
        return None                              # whole numbers
    logits = s["logits"].to(F64)
    slots, penalties = s["slots"].tolist(), s["penalties"].to(F64).tolist()
    for r in range(case["rows"]):
        row, count = logits[r], s["counts"][slots[r]].to(F64)
        held = _unpacked(s["seen"][slots[r]][None], vocab)[0].nonzero()[:, 0]
        z, n = row[held], count[held]
        divisor, presence, frequency = penalties[r]
        z = torch.where(z > 0, z / divisor, z * divisor)
        row[held] = z - torch.where(n > 0, presence, 0.0) - frequency * n
        if s["bias"] is not None:
            first, last = s["bias"][0][r:r + 2].tolist()
            row.index_add_(0, s["bias"][1][first:last].long(), s["bias"][2][first:last].to(F64))
        if s["masks"] is not None and s["masks"][0][r] >= 0:
            row[~_unpacked(s["masks"][1][s["masks"][0][r]][None], vocab)[0]] = -math.inf
    return logits


def _exact_shared(case, s):
    heads, kv, dim, page, new = (case[k] for k in ("heads", "kv", "dim", "page", "new"))
    group = heads // kv
    out = torch.empty(s["out"].shape, dtype=F64, device=DEVICE)
    tables = s["tables"].tolist()
    for i, table in enumerate(tables):
        held = s["pages"][torch.tensor([p for p in table if p >= 0], device=DEVICE), 0].to(F64)    # [pages, 2, kv, page, dim]
        k, v = held.permute(1, 2, 0, 3, 4).reshape(2, kv, -1, dim)
        for t in range(i * new, (i + 1) * new):
            seen = int(s["positions"][t]) + 1
            q = s["qkv"][t, :heads * dim].to(F64).view(kv, group, dim)
            weights = torch.softmax(torch.einsum("kgd,ksd->kgs", q, k[:, :seen]) / math.sqrt(dim), -1)
            out[t] = torch.einsum("kgs,ksd->kgd", weights, v[:, :seen]).reshape(-1)
    return out
