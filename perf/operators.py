"""The operators of a delta-rule mixer and of forked requests, as cases that can be timed and checked.

Kinds of cases:

  prompt   the gated delta rule over portions of prompts: requests of several lengths, their states in slots
  token    the same rule for one new token per request, as a decode step runs it
  prep     the short causal convolution of q, k and v in front of the rule, and the rule's gates
  copy     blocks copied inside pools of equal blocks: pages and states of forked requests, compaction

Sizes are those of the hybrid designs' mixers at widths 2,048 and 4,096 (16 or 32 heads of 128), of the 1.5B
and 7B layer stacks for pages, and generic ones.  Everything is drawn from the seed on the device.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False
DEVICE = "cuda:0"
F64 = torch.float64
EPS = 1e-6                  # inside the root of the keys' and queries' length
PLAIN_CHUNK = 64
PREP_TOKENS = 64            # tokens of a tile of the convolution
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def _rule(name, kind, lengths, heads, share, dim, vdim, dtype):
    return {"name": name, "kind": kind, "lengths": " ".join(map(str, lengths)), "heads": heads, "share": share,
            "dim": dim, "vdim": vdim, "dtype": dtype}


RAGGED = (700, 1, 64, 333, 17, 128, 2, 511, 90, 256, 31, 5, 190)


def listed():
    return [
        # one long prompt in a single portion at width 4,096: the chain of states is all there is to do in parallel
        _rule("prompt_8192", "prompt", [8192], 32, 2, 128, 128, "bf16"),
        # four prompts of 2,048 tokens in one step at the same width
        _rule("prompts_4x2048", "prompt", [2048] * 4, 32, 1, 128, 128, "bf16"),
        # a mixed step of the scheduler: ends of prompts, short prompts, decoded tokens, at smaller heads
        _rule("portions_ragged", "prompt", RAGGED, 12, 1, 64, 64, "bf16"),
        # a prompt of the 32-bit path, values narrower than the keys
        _rule("prompt_f32_611", "prompt", [611], 8, 1, 128, 96, "f32"),
        # a single request's decoded token at width 2,048: latency
        _rule("token_1", "token", [1], 16, 1, 128, 128, "bf16"),
        # a decode step of 64 requests at width 4,096: the states' bytes
        _rule("token_64", "token", [1] * 64, 32, 2, 128, 128, "bf16"),
        # a decode step of the 32-bit path with an odd number of requests and heads of another shape
        _rule("token_f32_33", "token", [1] * 33, 6, 1, 96, 160, "f32"),
        # the convolution in front of a 4,096-token step: q and k of 16 heads, v of 32
        {"name": "prep_4096", "kind": "prep", "lengths": "2048 1500 548", "channels": 8192, "heads": 32, "taps": 4,
         "extra": 4096, "dtype": "bf16"},
        # the same for a decode step of 24 requests
        {"name": "prep_tokens_24", "kind": "prep", "lengths": " ".join(["1"] * 24), "channels": 6144, "heads": 16,
         "taps": 4, "extra": 2048, "dtype": "bf16"},
        # one request of a 7B stack forked once: its last page
        {"name": "fork_page", "kind": "copy", "buffers": 1, "blocks": 48, "elements": 28 * 2 * 4 * 16 * 128, "sources": 1,
         "copies": 1, "dtype": "bf16"},
        # a hybrid of 24 delta-rule layers at width 2,048: the states of one request for eight continuations
        {"name": "fork_states", "kind": "copy", "buffers": 24, "blocks": 16, "elements": 16 * 128 * 128, "sources": 1,
         "copies": 8, "dtype": "f32"},
        # compaction of a pool of the 1.5B stack's pages
        {"name": "compact_pages", "kind": "copy", "buffers": 1, "blocks": 1600, "elements": 28 * 2 * 2 * 16 * 128,
         "sources": 600, "copies": 1, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "token", "token", "prep", "copy"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "copy":
        elements = 8 * _log_int(rng, 400, 60000)
        buffers = rng.choice([1, 1, 2, 7, 24])
        copies = rng.choice([1, 1, 2, 5])
        most = int(3.2e8 / (elements * buffers * DTYPES[dtype].itemsize * (copies + 1)))
        sources = _log_int(rng, 1, max(1, min(1000, most)))
        return {"kind": kind, "buffers": buffers, "blocks": sources * (copies + 1) + rng.randint(0, 20),
                "elements": elements, "sources": sources, "copies": copies, "dtype": dtype}
    if kind == "prep":
        requests = _log_int(rng, 1, 40)
        tokens = max(requests, _log_int(rng, 1, 4096))
        return {"kind": kind, "lengths": _cut(rng, tokens, requests), "channels": 16 * _log_int(rng, 6, 512) + 8,
                "heads": _log_int(rng, 2, 32), "taps": rng.choice([2, 3, 4, 4]), "extra": 8 * rng.randint(0, 256),
                "dtype": dtype}
    dim = rng.choice([128, 128, 64, 64, 96, 32, 80])
    vdim = rng.choice([128, 128, 64, 64, 96, 160, 48])
    share = rng.choice([1, 1, 2, 4])
    heads = share * max(1, _log_int(rng, 2, 22) // share)
    if kind == "token":
        requests = _log_int(rng, 1, max(1, min(200, int(64 * 32 * 16384 / (heads * dim * vdim)))))
        lengths = " ".join(["1"] * requests)
    else:
        tokens = _log_int(rng, 20, min(8192, int(0.5 * 8192 * 32 * 16384 / (heads * dim * vdim))))
        lengths = _cut(rng, tokens, min(tokens, _log_int(rng, 1, 20)))
    return {"kind": kind, "lengths": lengths, "heads": heads, "share": share, "dim": dim, "vdim": vdim, "dtype": dtype}


def _cut(rng, tokens, requests):
    """`tokens` in `requests` uneven pieces of one at least, as text."""
    places = sorted(rng.sample(range(1, tokens), requests - 1)) if requests > 1 else []
    return " ".join(str(b - a) for a, b in zip([0] + places, places + [tokens]))


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


# ----------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _requests(lengths, gen):
    """The lists of a step and its requests' slots (in no order, two slots more than requests)."""
    starts = [0]
    for n in lengths[:-1]:
        starts.append(starts[-1] + n)
    slots = torch.randperm(len(lengths) + 2, generator=gen, device=DEVICE)[:len(lengths)].to(torch.int32)
    return {"qstart": _ints(starts), "qlen": _ints(lengths), "slots": slots, "lengths": lengths}


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device=DEVICE).normal_(mean, std, generator=gen)

    if case["kind"] == "copy":
        buffers = [normal(case["blocks"], case["elements"]).to(dtype) for _ in range(case["buffers"])]
        order = torch.randperm(case["blocks"], generator=gen, device=DEVICE).to(torch.int32)
        n = case["sources"] * case["copies"]
        src = order[:case["sources"]].repeat_interleave(case["copies"])
        moves = torch.stack([src, order[case["sources"]:case["sources"] + n]], 1).contiguous()
        return {"case": case, "buffers": buffers, "moves": moves, "error": _ints([0])}
    lengths = _lengths(case)
    tokens, heads = sum(lengths), case["heads"]
    state = dict(_requests(lengths, gen), case=case, error=_ints([0]))
    items = len(lengths)
    if case["kind"] == "prep":
        channels, taps = case["channels"], case["taps"]
        width = -(-(channels + case["extra"] + 2 * heads) // 8) * 8
        tiles = [(i, r) for i, n in enumerate(lengths) for r in range(0, n, PREP_TOKENS)]
        state.update(
            proj=normal(tokens, width).to(dtype), tails=normal(items + 2, (taps - 1) * channels),
            conv=normal(taps, channels, std=0.5), a_log=torch.log(1 + 15 * torch.rand(heads, generator=gen, device=DEVICE)),
            dt_bias=normal(heads, std=1.0, mean=-3.0), seg_item=_ints([i for i, _ in tiles]),
            seg_row0=_ints([r for _, r in tiles]),
            act=torch.empty(tokens, channels, dtype=dtype, device=DEVICE),
            log_decay=torch.empty(tokens, heads, device=DEVICE), beta=torch.empty(tokens, heads, device=DEVICE))
        return state
    dim, vdim, narrow = case["dim"], case["vdim"], case["heads"] // case["share"]
    width = 2 * narrow * dim + heads * vdim
    state.update(
        qkv=F.silu(normal(tokens, width)).to(dtype),
        # decays between nearly one and e^-2 or so a token, as exp(-exp(a_log) * softplus(.)) gives them
        log_decay=-torch.exp(normal(tokens, heads, std=1.5, mean=-3.0)), beta=torch.sigmoid(normal(tokens, heads)),
        state=normal(items + 2, heads * dim * vdim, std=0.1), out=torch.empty(tokens, heads * vdim, device=DEVICE))
    return state


# --------------------------------------------------------------------------------------- one pass
def run(s):
    return {"prompt": _run_rule, "token": _run_rule, "prep": _run_prep, "copy": _run_copy}[s["case"]["kind"]](s)


def _run_rule(s):
    c = s["case"]
    heads, dim, vdim, share = c["heads"], c["dim"], c["vdim"], c["share"]
    qk = heads // share * dim
    if own:
        from from_scratch_inference_engine_b200.kernels import ops
        ops.gated_delta_rule(s["qkv"], 0, qk, 2 * qk, s["log_decay"], s["beta"], s["qstart"], s["qlen"], s["slots"],
                             len(s["lengths"]), s["state"], s["out"], heads, dim, vdim, share=share, eps=EPS,
                             longest=max(s["lengths"]))
        return {"out": s["out"], "state": s["state"]}
    rows, seen = _rows(s)
    slots = s["slots"].long()

    def by_head(x, count, width):                     # [requests, heads, tokens, width], zeros behind the end
        x = x.view(-1, count, width)[rows] * seen[..., None, None]
        return x.permute(0, 2, 1, 3).repeat_interleave(heads // count, 1)
    qkv = s["qkv"].float()
    q = by_head(qkv[:, :qk], heads // share, dim)
    k = by_head(qkv[:, qk:2 * qk], heads // share, dim)
    v = by_head(qkv[:, 2 * qk:], heads, vdim)
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + EPS) * dim ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + EPS)
    decay, beta = (by_head(s[name], heads, 1)[..., 0] for name in ("log_decay", "beta"))
    old = s["state"][slots].view(-1, heads, dim, vdim)
    if max(s["lengths"]) == 1:
        a, b, k0, q0 = decay.exp()[..., None], beta[..., None], k.squeeze(2), q.squeeze(2)
        u = b.squeeze(-1) * (v.squeeze(2) - a.squeeze(-1) * (old * k0[..., None]).sum(2))
        new = a[..., None].squeeze(2) * old + k0[..., None] * u[:, :, None]
        o = (new * q0[..., None]).sum(2)[:, None]
    else:
        o, new = _chunked(q, k, v, decay, beta, old)
        o = o.permute(0, 2, 1, 3)
    s["out"][rows[seen]] = o[seen].reshape(-1, heads * vdim)
    s["state"][slots] = new.reshape(len(slots), -1)
    return {"out": s["out"], "state": s["state"]}


def _rows(s):
    """[requests, longest]: the row of each request's r-th token, and whether there is one."""
    r = torch.arange(max(s["lengths"]), device=DEVICE)
    seen = r < s["qlen"][:, None]
    return torch.where(seen, s["qstart"][:, None].long() + r, 0), seen


def _chunked(q, k, v, decay, beta, state):
    """The rule in chunks of tokens: inside a chunk a triangular system, from chunk to chunk the state."""
    batch, heads, tokens, _ = q.shape
    size = min(PLAIN_CHUNK, tokens)
    count = -(-tokens // size)

    def cut(x):
        x = F.pad(x, (0, 0, 0, count * size - tokens)) if x.dim() == 4 else F.pad(x, (0, count * size - tokens))
        return x.view(batch, heads, count, size, *x.shape[3:])
    q, k, v, beta, total = cut(q), cut(k), cut(v), cut(beta)[..., None], cut(decay).cumsum(-1)
    lower = torch.ones(size, size, dtype=torch.bool, device=DEVICE).tril()
    between = torch.where(lower, total[..., :, None] - total[..., None, :], -math.inf).exp()
    total = total[..., None]
    a = (beta * (k @ k.mT) * between).tril(-1)
    inverse = torch.eye(size, device=DEVICE).expand_as(a).clone()
    for i in range(1, size):
        inverse[..., i, :i] = -(a[..., i, None, :i] @ inverse[..., :i, :i])[..., 0, :]
    given, taken = inverse @ (beta * v), inverse @ (beta * total.exp() * k)
    seen, q, last = (q @ k.mT) * between, q * total.exp(), total[..., -1:, :]
    k, last = k * (last - total).exp(), last.exp()
    outs = []
    for n in range(count):
        u = given[:, :, n] - taken[:, :, n] @ state
        outs.append(q[:, :, n] @ state + seen[:, :, n] @ u)
        state = last[:, :, n] * state + k[:, :, n].mT @ u
    return torch.stack(outs, 2).reshape(batch, heads, count * size, -1)[:, :, :tokens], state


def _run_prep(s):
    c = s["case"]
    channels, heads, taps = c["channels"], c["heads"], c["taps"]
    a_off = channels + c["extra"]
    if own:
        from from_scratch_inference_engine_b200.kernels import ops
        ops.delta_prep(s["proj"], 0, a_off, a_off + heads, s["qstart"], s["qlen"], s["slots"], len(s["lengths"]),
                       s["seg_item"], s["seg_row0"], s["seg_item"].numel(), PREP_TOKENS, s["tails"], 0, s["conv"],
                       s["a_log"], s["dt_bias"], s["act"], s["log_decay"], s["beta"])
        return {"act": s["act"], "log_decay": s["log_decay"], "beta": s["beta"], "tails": s["tails"]}
    rows, seen = _rows(s)
    slots = s["slots"].long()
    proj = s["proj"].float()
    before = s["tails"][slots].view(-1, taps - 1, channels)
    u = torch.cat([before, proj[:, :channels][rows]], 1)
    longest = rows.shape[1]
    act = F.silu(sum(s["conv"][j] * u[:, j:j + longest] for j in range(taps)))
    s["act"][rows[seen]] = act[seen].to(s["act"].dtype)
    last = s["qlen"][:, None].long() + torch.arange(taps - 1, device=DEVICE)
    s["tails"][slots] = u.gather(1, last[..., None].expand(-1, -1, channels)).reshape(len(slots), -1)
    s["log_decay"].copy_(-s["a_log"].exp() * F.softplus(proj[:, a_off:a_off + heads] + s["dt_bias"]))
    s["beta"].copy_(torch.sigmoid(proj[:, a_off + heads:a_off + 2 * heads]))
    return {"act": s["act"], "log_decay": s["log_decay"], "beta": s["beta"], "tails": s["tails"]}


def _run_copy(s):
    if own:
        from from_scratch_inference_engine_b200.kernels import ops
        ops.copy_blocks(s["buffers"], s["moves"], s["error"])
        return s["buffers"]
    src, dst = s["moves"].long().unbind(1)
    for buffer in s["buffers"]:
        buffer[dst] = buffer[src]
    return s["buffers"]


# ------------------------------------------------------------------------------- bytes, operations
def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "copy":
        blocks = case["sources"] * (1 + case["copies"])
        return {"bytes": blocks * case["buffers"] * case["elements"] * size + 8 * case["sources"] * case["copies"], "flops": 0}
    lengths = _lengths(case)
    tokens, heads, items = sum(lengths), case["heads"], len(lengths)
    if case["kind"] == "prep":
        channels, taps = case["channels"], case["taps"]
        return {"bytes": tokens * (2 * channels * size + heads * (2 * size + 8)) + 8 * items * (taps - 1) * channels
                + 4 * taps * channels, "flops": tokens * channels * (2 * taps + 4)}
    dim, vdim = case["dim"], case["vdim"]
    row = 2 * (heads // case["share"]) * dim * size + heads * vdim * (size + 4) + 8 * heads
    return {"bytes": tokens * row + 8 * items * heads * dim * vdim, "flops": 6 * tokens * heads * dim * vdim}


# -------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        src, dst = s["moves"].long().unbind(1)
        return [b.double().index_copy(0, dst, b.double().index_select(0, src)) for b in s["buffers"]]
    lengths, heads = _lengths(case), case["heads"]
    starts = [sum(lengths[:i]) for i in range(len(lengths))]
    slots = s["slots"].tolist()
    if case["kind"] == "prep":
        return _exact_prep(case, s, lengths, starts, slots)
    dim, vdim, share = case["dim"], case["vdim"], case["share"]
    narrow = heads // share
    qkv = s["qkv"].to(F64)
    q = qkv[:, :narrow * dim].reshape(-1, narrow, dim).repeat_interleave(share, 1)
    k = qkv[:, narrow * dim:2 * narrow * dim].reshape(-1, narrow, dim).repeat_interleave(share, 1)
    v = qkv[:, 2 * narrow * dim:].reshape(-1, heads, vdim)
    q = q / torch.sqrt(q.square().sum(-1, keepdim=True) + EPS) / math.sqrt(dim)
    k = k / torch.sqrt(k.square().sum(-1, keepdim=True) + EPS)
    a, b = torch.exp(s["log_decay"].to(F64)), s["beta"].to(F64)
    state = s["state"].to(F64)
    out = torch.zeros(len(qkv), heads, vdim, dtype=F64, device=DEVICE)
    # token by token, all requests that still have one side by side
    for r in range(max(lengths)):
        left = [i for i, n in enumerate(lengths) if n > r]
        rows = torch.tensor([starts[i] + r for i in left], device=DEVICE)
        at = torch.tensor([slots[i] for i in left], device=DEVICE)
        held = state[at].view(-1, heads, dim, vdim) * a[rows][..., None, None]
        u = b[rows][..., None] * (v[rows] - torch.einsum("ihdv,ihd->ihv", held, k[rows]))
        held = held + k[rows][..., None] * u[:, :, None]
        out[rows] = torch.einsum("ihdv,ihd->ihv", held, q[rows])
        state[at] = held.reshape(len(left), -1)
    return {"out": out.reshape(len(qkv), -1), "state": state}


def _exact_prep(case, s, lengths, starts, slots):
    channels, heads, taps = case["channels"], case["heads"], case["taps"]
    a_off = channels + case["extra"]
    proj, tails, w = s["proj"].to(F64), s["tails"].to(F64).view(-1, taps - 1, channels), s["conv"].to(F64)
    act = torch.empty(len(proj), channels, dtype=F64, device=DEVICE)
    for n, start, slot in zip(lengths, starts, slots):
        u = torch.cat([tails[slot], proj[start:start + n, :channels]])
        c = torch.zeros(n, channels, dtype=F64, device=DEVICE)
        for j in range(taps):
            c += w[j] * u[j:j + n]
        act[start:start + n] = c / (1 + torch.exp(-c))
        tails[slot] = u[n:]
    step = torch.log1p(torch.exp(proj[:, a_off:a_off + heads] + s["dt_bias"].to(F64)))
    return {"act": act, "log_decay": -torch.exp(s["a_log"].to(F64)) * step,
            "beta": 1 / (1 + torch.exp(-proj[:, a_off + heads:a_off + 2 * heads])), "tails": tails.view(len(tails), -1)}
