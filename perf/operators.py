"""What the operators around a cache of bounded length and the scoring of given tokens are measured on.

    mass      attention_mass: what every cached key has drawn of the queries' attention, added up beside the keys
    select    evict_select: which places of the cache stay, by that sum
    compact   cache_compact: the kept places' keys, values and sums move to the front of the requests' pages
    logprobs  token_logprobs: log probability of given tokens, entropy and the likeliest tokens of rows of logits

`own` false: the plain form, elementary torch operations in 32 bits; true: the calls that the engine and its sampler make.
"""
import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

PAGE = 16
# (heads, kv heads, head size, layers, vocabulary) of the family's members that the benchmark names
MODELS = {"0.5b": (14, 2, 64, 24, 151936), "1.5b": (12, 2, 128, 28, 151936), "7b": (28, 4, 128, 28, 152064), "32b": (40, 8, 128, 64, 152064)}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one layer of one short chat on the smallest member: launches and latency
        dict(name="mass_decode_1_0p5b", kind="mass", model="0.5b", dtype="bf16", prompts=0, cached=0, tokens=0, requests=1, shortest=300, longest=300),
        # a full batch that decodes, contexts of all lengths
        dict(name="mass_decode_64_1p5b", kind="mass", model="1.5b", dtype="bf16", prompts=0, cached=0, tokens=0, requests=64, shortest=100, longest=2001),
        # three long documents in the 32-bit path
        dict(name="mass_decode_3_32k_fp32", kind="mass", model="7b", dtype="fp32", prompts=0, cached=0, tokens=0, requests=3, shortest=20000, longest=32001),
        # the benchmark's prompt, whole
        dict(name="mass_prompt_2048_7b", kind="mass", model="7b", dtype="bf16", prompts=1, cached=0, tokens=2048, requests=0, shortest=0, longest=0),
        # a late portion of a long document beside requests that decode, an odd number of rows
        dict(name="mass_portion_32b", kind="mass", model="32b", dtype="bf16", prompts=1, cached=16000, tokens=1999, requests=5, shortest=50, longest=1500),
        # every layer of a batch of full contexts is cut to half
        dict(name="select_8_7b", kind="select", model="7b", layers=28, requests=8, shortest=2500, longest=4096, keep=2048, first=4, recent=512),
        # one long document, a few layers, cut to an eighth
        dict(name="select_1_32k", kind="select", model="32b", layers=8, requests=1, shortest=32001, longest=32001, keep=4000, first=4, recent=1000),
        # the same two cuts, carried out
        dict(name="compact_8_7b", kind="compact", model="7b", dtype="bf16", layers=28, requests=8, shortest=2500, longest=4096, keep=2048, first=4, recent=512),
        dict(name="compact_1_fp32", kind="compact", model="0.5b", dtype="fp32", layers=24, requests=1, shortest=701, longest=701, keep=400, first=4, recent=64),
        # the alternatives of one chat's next token
        dict(name="logprobs_1", kind="logprobs", rows=1, vocab=151936, top=5),
        # a full batch with twenty alternatives each
        dict(name="logprobs_64", kind="logprobs", rows=64, vocab=152064, top=20),
        # a prompt that is scored
        dict(name="logprobs_2047", kind="logprobs", rows=2047, vocab=151936, top=1),
    ]


def _spread(rng, low, high):
    """A whole number between the two, evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["mass", "mass", "mass", "select", "compact", "logprobs"])
    if kind == "logprobs":
        return dict(kind=kind, rows=_spread(rng, 1, 2000), vocab=rng.choice([32000, 32003, 151936, 152064]), top=rng.choice([0, 1, 5, 20, 32]))
    if kind == "mass":
        model, dtype = rng.choice(list(MODELS)), rng.choice(["bf16", "bf16", "bf16", "fp32"])
        case = dict(kind=kind, model=model, dtype=dtype, prompts=0, cached=0, tokens=0, requests=0, shortest=0, longest=0)
        if rng.random() < 0.5:
            n = _spread(rng, 1, 64)
            longest = _spread(rng, 2, min(32000, 65000 // n))
            return dict(case, requests=n, shortest=max(1, longest // rng.choice([1, 2, 8])), longest=longest)
        prompts = _spread(rng, 1, 8)
        most = 1000 if dtype == "fp32" else 2000
        case.update(prompts=prompts, tokens=_spread(rng, 2, most // prompts), cached=rng.choice([0, _spread(rng, 1, 8000 // prompts)]))
        if rng.random() < 0.5:
            case.update(requests=_spread(rng, 1, 16), shortest=20, longest=_spread(rng, 20, 2000))
        return case
    model = rng.choice(list(MODELS))
    n = _spread(rng, 1, 8)
    longest = _spread(rng, 40, 4096)
    keep = _spread(rng, 8, longest)
    case = dict(kind=kind, model=model, layers=rng.choice([1, 8, 24]), requests=n, shortest=max(1, longest // rng.choice([1, 2, 4])),
                longest=longest, keep=keep, first=rng.choice([0, 1, 4]), recent=rng.choice([0, keep // 4, keep // 2]))
    return dict(case, dtype=rng.choice(["bf16", "bf16", "fp32"])) if kind == "compact" else case


def lengths(case):
    """The requests' lengths, spread evenly from the shortest to the longest, in an order that mixes them."""
    n, low, high = case["requests"], case["shortest"], case["longest"]
    out = [low + (high - low) * i // max(1, n - 1) if n > 1 else high for i in range(n)]
    random.Random(7).shuffle(out)
    return out


def segments(case):
    """[(tokens of the step, cached length after it)] of a `mass` case: prompts of falling length, then single tokens."""
    p = case["prompts"]
    multi = [(max(2, case["tokens"] - i * case["tokens"] // (2 * p)), 0) for i in range(p)]
    return [(q, case["cached"] + q) for q, _ in multi] + [(1, n) for n in lengths(case)]


# ---------------------------------------------------------------------------------------------------------- inputs
def _tables(lens, g, device):
    """(block tables, number of pages): pages in a random order, a few that nobody holds between them."""
    blocks = [-(-n // PAGE) for n in lens]
    pages = sum(blocks) + 3
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    at = torch.tensor([0] + blocks, device=device).cumsum(0)[:-1, None] + torch.arange(max(blocks), device=device)
    held = torch.arange(max(blocks), device=device) < torch.tensor(blocks, device=device)[:, None]
    return torch.where(held, order[at.clamp(max=pages - 1)], -1).to(torch.int32).contiguous(), pages


def _drawn_mass(shape, g, device):
    """Sums as a long run leaves them: a few keys draw most of the attention, some none."""
    m = torch.exp(2.0 * torch.randn(shape, generator=g, device=device))
    return torch.where(torch.rand(shape, generator=g, device=device) < 0.05, 0.0, m)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    state = dict(case=case)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=device)
    if case["kind"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        # a language model's rows: wide, with some tokens far ahead; ids that are mostly likely ones
        x = torch.randn((n, v), generator=g, device=device) * 2.5
        x[torch.arange(n, device=device)[:, None], torch.randint(0, v, (n, 16), generator=g, device=device)] += 12.0 * torch.rand((n, 16), generator=g, device=device)
        ids = torch.where(torch.rand(n, generator=g, device=device) < 0.5, x.argmax(1), torch.randint(0, v, (n,), generator=g, device=device))
        state.update(logits=x, ids=ids.to(torch.int32))
        return state
    nh, nkv, dh, _, _ = MODELS[case["model"]]
    if case["kind"] == "mass":
        segs = segments(case)
        q_len, ctx = [q for q, _ in segs], [c for _, c in segs]
        t, dt = sum(q_len), TYPES[case["dtype"]]
        table, pages = _tables(ctx, g, device)
        k = torch.randn((pages, nkv, PAGE, dh), generator=g, device=device) * torch.exp(0.3 * torch.randn((pages, nkv, PAGE, 1), generator=g, device=device))
        qkv = torch.randn((t, (nh + 2 * nkv) * dh), generator=g, device=device) * 1.5
        singles = [c for q, c in segs if q == 1]
        q_start = [sum(q_len[:i]) for i in range(len(q_len))]
        # the step's batch as the engine lays it out once for all layers
        host = {"host_q_start": q_start, "host_q_len": q_len, "host_ctx_len": ctx}
        meta = SimpleNamespace(block_table=table, max_blocks=table.shape[1], seg_of_token=ints([i for i, q in enumerate(q_len) for _ in range(q)]),
                               q_start=ints(q_start), q_len=ints(q_len), ctx_len=ints(ctx), num_segments=len(segs), num_tokens=t,
                               max_q_len=max(q_len), max_ctx_len=max(ctx), num_single=len(singles), num_multi=t - len(singles),
                               max_single_ctx=max(singles, default=0), padded=False, extra={}, **{n: np.array(v, dtype=np.int32) for n, v in host.items()})
        # (sums of a few steps: what this one adds is not lost beside them)
        state.update(qkv=qkv.to(dt), k=k.to(dt), mass=1e-3 * _drawn_mass((pages, nkv, PAGE, 1), g, device), meta=meta)
        return state
    lens = lengths(case)
    table, pages = _tables(lens, g, device)
    layers = case["layers"]
    state.update(table=table, lens=ints(lens), keep=ints([case["keep"]] * len(lens)), mass=_drawn_mass((layers, pages, nkv, PAGE, 1), g, device))
    if case["kind"] == "compact":
        dt = TYPES[case["dtype"]]
        state["k"], state["v"] = (torch.randn((layers, pages, nkv, PAGE, dh), generator=g, device=device).to(dt) for _ in range(2))
        state["kept"] = _select(state)
    return state


# -------------------------------------------------------------------------------------------------- the plain forms
def _gathered(x, table):
    """Rows [..., requests, heads, places, size] of x [..., pages, heads, page, size]; places of pages that are not there hold anything."""
    p = table.long().clamp(min=0)
    rows = x[..., p, :, :, :]                                    # [..., n, blocks, heads, page, size]
    rows = rows.transpose(-4, -3)
    return rows.flatten(-3, -2)


def _mass_of(state, part, mq, places):
    """The segments `part` of the batch: up to mq queries each, up to so many places of the cache."""
    case, meta = state["case"], state["meta"]
    nh, nkv, dh, _, _ = MODELS[case["model"]]
    qkv, mass, table = state["qkv"], state["mass"], meta.block_table[part, :-(-places // PAGE)]
    i, t = torch.arange(mq, device=qkv.device), torch.arange(table.shape[1] * PAGE, device=qkv.device)
    q_start, q_len, ctx = (x[part].long() for x in (meta.q_start, meta.q_len, meta.ctx_len))
    n, places = len(ctx), len(t)
    rows = (q_start[:, None] + i).clamp(max=meta.num_tokens - 1)                                    # [n, mq]
    q = qkv[rows, :nh * dh].float().view(n, mq, nkv, nh // nkv, dh).permute(0, 2, 3, 1, 4).reshape(n, nkv, nh // nkv * mq, dh)
    keys = _gathered(state["k"], table).float()                                                     # [n, nkv, places, dh]
    s = torch.matmul(q * (1.0 / math.sqrt(dh)), keys.transpose(-1, -2).contiguous()).view(n, nkv, nh // nkv, mq, places)
    at = ctx[:, None] - q_len[:, None] + i                                                          # where each query stands
    seen = (t <= at[:, :, None]) & (i < q_len[:, None])[:, :, None]                                 # [n, mq, places]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    drawn = (e / e.sum(-1, keepdim=True).clamp(min=1e-30)).sum((2, 3))                              # [n, nkv, places]
    pages = table.long().clamp(min=0).repeat_interleave(PAGE, 1)                                    # [n, places]
    old = mass[pages, :, t % PAGE, 0].transpose(1, 2)                                               # [n, nkv, places]
    new = torch.where((t >= (ctx - q_len)[:, None])[:, None], drawn, old + drawn)
    r, c = (t < ctx[:, None]).nonzero(as_tuple=True)
    mass[pages[r, c], :, c % PAGE, 0] = new.transpose(1, 2)[r, c]


def _mass(state):
    meta, p = state["meta"], state["case"]["prompts"]
    if p:
        _mass_of(state, slice(0, p), meta.max_q_len, int(meta.host_ctx_len[:p].max()))
    if meta.num_single:
        _mass_of(state, slice(p, None), 1, meta.max_single_ctx)
    return state["mass"]


def _select(state):
    case, lens, keep = state["case"], state["lens"].long(), state["keep"].long()
    mass = _gathered(state["mass"], state["table"])[..., 0]                                         # [layers, n, heads, places]
    t = torch.arange(mass.shape[-1], device=mass.device)
    keep = torch.minimum(keep, lens)
    recent = keep.clamp(max=case["recent"])
    first = (keep - recent).clamp(max=case["first"])
    always = (t < first[:, None]) | ((t >= (lens - recent)[:, None]) & (t < lens[:, None]))
    m = mass.masked_fill(always[:, None], float("inf")).masked_fill((t >= lens[:, None])[:, None], float("-inf"))
    order = torch.sort(m, dim=-1, descending=True, stable=True).indices[..., :case["keep"]]
    rank = torch.arange(order.shape[-1], device=mass.device)
    order = order.masked_fill((rank >= keep[:, None])[:, None], 1 << 40)
    order = torch.sort(order, -1).values
    out = torch.full((*order.shape[:-1], case["keep"]), -1, dtype=torch.int32, device=mass.device)
    out[..., :order.shape[-1]] = torch.where(order < 1 << 40, order, -1).to(torch.int32)
    return out


def _compact(state):
    kept, table = state["kept"].long(), state["table"].long()
    layer, r, h, j = (kept >= 0).nonzero(as_tuple=True)
    src = kept[layer, r, h, j]
    from_page, to_page = table[r, src // PAGE], table[r, j // PAGE]
    return {name: state[name].index_put_((layer, to_page, h, j % PAGE), state[name][layer, from_page, h, src % PAGE]) for name in ("k", "v", "mass")}


def _logprobs(state):
    x, ids, top = state["logits"], state["ids"].long(), state["case"]["top"]
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    out = {"logprobs": (d.gather(1, ids[:, None]) - log_total)[:, 0], "entropy": (log_total - (e * d).sum(1, keepdim=True) / total)[:, 0]}
    if top:
        values, at = torch.sort(x, dim=1, descending=True, stable=True)
        out["top_ids"] = at[:, :top].to(torch.int32)
        out["top_logprobs"] = values[:, :top] - x.amax(1, keepdim=True) - log_total
    return out


# ---------------------------------------------------------------------------------------- the framework's own calls
def _own(state):
    from litinfer_amd.engine.workspace import Workspace
    from litinfer_amd.kernels import ops
    case = state["case"]
    if case["kind"] == "logprobs":
        x = state["logits"]
        n, top = x.shape[0], case["top"]
        out = {name: torch.empty(n, dtype=torch.float32, device=x.device) for name in ("logprobs", "entropy")}
        if top:
            out["top_ids"] = torch.empty((n, top), dtype=torch.int32, device=x.device)
            out["top_logprobs"] = torch.empty((n, top), dtype=torch.float32, device=x.device)
        ops.token_logprobs(x, state["ids"], out["logprobs"], out["entropy"], out.get("top_ids"), out.get("top_logprobs"))
        return out
    if case["kind"] == "mass":
        nh, nkv, dh, _, _ = MODELS[case["model"]]
        if "ws" not in state:
            state["ws"] = Workspace(state["qkv"].device)         # (the engine's, which lives as long as it)
        ops.attention_mass(state["qkv"], state["mass"], state["k"], state["meta"], nh, nkv, dh, PAGE, 1.0 / math.sqrt(dh), ws=state["ws"])
        return state["mass"]
    if case["kind"] == "select":
        mass, table = state["mass"], state["table"]
        out = torch.empty((mass.shape[0], table.shape[0], mass.shape[2], case["keep"]), dtype=torch.int32, device=mass.device)
        ops.evict_select(mass, table, state["lens"], state["keep"], case["first"], case["recent"], out)
        return out
    names = ("k", "v", "mass")
    ops.cache_compact([state[n] for n in names], state["table"], state["kept"])
    return {n: state[n] for n in names}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "mass":
        return _mass(state)
    if kind == "select":
        return _select(state)
    return _compact(state) if kind == "compact" else _logprobs(state)


# ------------------------------------------------------------------------------------------------------- the floors
def work(case):
    if case["kind"] == "logprobs":
        n, v, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4 * n * v + n * (12 + 8 * top), "flops": 5 * n * v}
    nh, nkv, dh, _, _ = MODELS[case["model"]]
    if case["kind"] == "mass":
        es = 2 if case["dtype"] == "bf16" else 4
        segs = segments(case)
        pairs = sum(q * (c - q) + q * (q + 1) // 2 for q, c in segs)
        keys = sum(c for _, c in segs)
        fresh = sum(q for q, _ in segs)
        return {"bytes": keys * nkv * dh * es + fresh * nh * dh * es + (2 * keys - fresh) * nkv * 4, "flops": 2 * pairs * nh * dh}
    lens, layers = lengths(case), case["layers"]
    kept = sum(min(n, case["keep"]) for n in lens)
    if case["kind"] == "select":
        return {"bytes": 4 * layers * nkv * (sum(lens) + case["keep"] * len(lens)), "flops": layers * nkv * sum(lens)}
    es = 2 if case["dtype"] == "bf16" else 4
    # (the rows in front, and all rows of a request that is not cut, stay where they are)
    moved = sum(case["keep"] - case["first"] for n in lens if n > case["keep"])
    return {"bytes": layers * nkv * (4 * kept + max(1, moved) * 2 * (2 * dh * es + 4)), "flops": 0}


# -------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "logprobs":
        x, ids = state["logits"], state["ids"].long()
        lp, ent, tops = [], [], []
        for a in range(0, x.shape[0], 256):                          # (a part of the rows at a time: 64 bits of all of them take room)
            y = torch.log_softmax(x[a:a + 256].double(), 1)
            lp.append(y.gather(1, ids[a:a + 256, None])[:, 0])
            p = torch.exp(y)
            ent.append(-(p * y.masked_fill(p == 0, 0.0)).sum(1))
            tops.append(y.sort(1, descending=True).values[:, :case["top"]])
        out = {"logprobs": torch.cat(lp), "entropy": torch.cat(ent)}
        if case["top"]:
            out.update(top_ids=None, top_logprobs=torch.cat(tops))
        return out
    if case["kind"] == "select":
        return None                                                  # (whole numbers)
    if case["kind"] == "compact":
        out = {}
        for name in ("k", "v", "mass"):
            x = out[name] = state[name].double()
            for layer in range(x.shape[0]):
                for r, n in enumerate(lengths(case)):
                    page, off = state["table"][r].long().repeat_interleave(PAGE)[:n], torch.arange(n, device=x.device) % PAGE
                    for h in range(x.shape[2]):
                        src = state["kept"][layer, r, h][:min(n, case["keep"])].long()
                        x[layer, page[:len(src)], h, off[:len(src)]] = x[layer, page, h, off][src]
        return out
    nh, nkv, dh, _, _ = MODELS[case["model"]]
    mass, meta = state["mass"].double(), state["meta"]
    rep, at = nh // nkv, 0
    for r, (q, c) in enumerate(segments(case)):
        slots = torch.arange(c, device=mass.device)
        page = meta.block_table[r].long()[slots // PAGE]
        where = slots[None, :] <= torch.arange(c - q, c, device=mass.device)[:, None]
        for h in range(nkv):
            keys = state["k"][page, h, slots % PAGE].double()
            total = torch.zeros(c, dtype=torch.float64, device=mass.device)
            for m in range(h * rep, (h + 1) * rep):
                s = state["qkv"][at:at + q, m * dh:(m + 1) * dh].double() @ keys.t() / math.sqrt(dh)
                total += torch.softmax(s.masked_fill(~where, float("-inf")), 1).sum(0)
            old = mass[page, h, slots % PAGE, 0]
            mass[page, h, slots % PAGE, 0] = torch.where(slots >= c - q, total, old + total)
        at += q
    return mass
