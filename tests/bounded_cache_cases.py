"""Plain forms in 64 bits of the operators around a cache of bounded length and of token_logprobs, and inputs at the sizes where
they can go wrong."""
import math
from types import SimpleNamespace

import numpy as np
import torch


def batch(segs, page_size, device, seed=0, spare=3, holes=()):
    """A step's batch as the kernels take it: `segs` [(tokens of the step, cached length after it)], pages in a random order, tables
    padded with -1; `holes` (request, block) entries of the tables are -1 too."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-c // page_size) for _, c in segs]
    pages = sum(blocks) + spare
    order = torch.randperm(pages, generator=g).tolist()
    width = max(blocks) + 1
    table = torch.full((len(segs), width), -1, dtype=torch.int32)
    for r, b in enumerate(blocks):
        for j in range(b):
            table[r, j] = order.pop()
    for r, j in holes:
        table[r, j] = -1
    q_len = [q for q, _ in segs]
    ctx = [c for _, c in segs]
    start = np.cumsum([0] + q_len)[:-1]
    singles = [c for q, c in segs if q == 1]

    def ints(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32).to(device)
    return SimpleNamespace(block_table=table.to(device), max_blocks=width, seg_of_token=ints(np.repeat(np.arange(len(segs)), q_len)), q_start=ints(start),
                           q_len=ints(q_len), ctx_len=ints(ctx), num_segments=len(segs), num_tokens=sum(q_len), max_q_len=max(q_len),
                           max_ctx_len=max(ctx), num_single=len(singles), num_multi=sum(q_len) - len(singles), max_single_ctx=max(singles, default=0),
                           padded=False, extra={}, host_q_start=np.asarray(start, dtype=np.int32), host_q_len=np.asarray(q_len, dtype=np.int32),
                           host_ctx_len=np.asarray(ctx, dtype=np.int32)), pages


def plain_mass(qkv, mass, k, meta, nh, nkv, dh, page_size, scale, fresh=True):
    """attention_mass in 64 bits on the CPU: what `mass` holds afterwards (float64)."""
    qkv, k, table = qkv.cpu().double(), k.cpu().double(), meta.block_table.cpu().long()
    out = mass.cpu().double().clone()
    for r in range(meta.num_segments):
        q, c, at = int(meta.host_q_len[r]), int(meta.host_ctx_len[r]), int(meta.host_q_start[r])
        t = torch.arange(c)
        page = table[r, t // page_size]
        there = page >= 0
        seen = (t[None, :] <= torch.arange(c - q, c)[:, None]) & there[None, :]
        for g in range(nkv):
            keys = k[page.clamp(min=0), g, t % page_size]
            drawn = torch.zeros(c, dtype=torch.float64)
            for h in range(g * nh // nkv, (g + 1) * nh // nkv):
                s = (qkv[at:at + q, h * dh:(h + 1) * dh] @ keys.T * scale).masked_fill(~seen, -math.inf)
                drawn += torch.nan_to_num(torch.softmax(s, 1), nan=0.0).sum(0) if not there.all() else torch.softmax(s, 1).sum(0)
            new = torch.where((t >= c - q) & bool(fresh), drawn, out[page.clamp(min=0), g, t % page_size, 0] + drawn)
            out[page[there], g, t[there] % page_size, 0] = new[there]
    return out


def plain_select(mass, table, lens, keep, first, recent, room):
    """evict_select, one list at a time."""
    mass, table = mass.cpu(), table.cpu().long()
    entries, _, nkv, page_size, _ = mass.shape
    out = torch.full((entries, len(lens), nkv, room), -1, dtype=torch.int32)
    for e in range(entries):
        for r, (n, want) in enumerate(zip(lens, keep)):
            want = min(want, n, room)
            last = min(recent, want)
            front = min(first, want - last)
            for g in range(nkv):
                vals = [float(mass[e, table[r, t // page_size], g, t % page_size, 0]) if table[r, t // page_size] >= 0 else math.nan for t in range(n)]
                middle = sorted(range(front, n - last), key=lambda t: (-math.inf if math.isnan(vals[t]) else vals[t], not math.isnan(vals[t]), -t), reverse=True)
                places = sorted(list(range(front)) + middle[:want - front - last] + list(range(n - last, n)))
                out[e, r, g, :len(places)] = torch.tensor(places, dtype=torch.int32)
    return out


def plain_compact(tensors, table, kept):
    """cache_compact, a row at a time; new tensors on the CPU."""
    table, kept = table.cpu().long(), kept.cpu()
    out = [t.cpu().clone() for t in tensors]
    page_size = tensors[0].shape[3]
    for t, src in zip(out, [t.cpu() for t in tensors]):
        for e in range(kept.shape[0]):
            for r in range(kept.shape[1]):
                for g in range(kept.shape[2]):
                    for j, p in enumerate(kept[e, r, g].tolist()):
                        if p < 0:
                            break
                        t[e, table[r, j // page_size], g, j % page_size] = src[e, table[r, p // page_size], g, p % page_size]
    return out


def plain_logprobs(x, ids, top):
    """token_logprobs in 64 bits: (log probabilities, entropies, top ids, top log probabilities)."""
    y = torch.log_softmax(x.cpu().double(), 1)
    p = torch.exp(y)
    entropy = -(p * y.masked_fill(p == 0, 0.0)).sum(1)
    ids = ids.cpu().long()
    inside = (ids >= 0) & (ids < x.shape[1])
    lp = torch.where(inside, y.gather(1, ids.clamp(0, x.shape[1] - 1)[:, None])[:, 0], math.nan)
    order = torch.sort(x.cpu().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf), dim=1, descending=True, stable=True).indices[:, :top]
    return lp, entropy, order.to(torch.int32), y.gather(1, order)


# ------------------------------------------------------------------------------------ stand-ins for the kernels (CPU tests)
def attention_mass(qkv, mass, k, meta, nh, nkv, dh, page_size, scale, fresh=True, ws=None):
    mass.copy_(plain_mass(qkv, mass, k, meta, nh, nkv, dh, page_size, scale, fresh).float())


def evict_select(mass, block_table, lens, keep, first, recent, out):
    out.copy_(plain_select(mass, block_table, lens.tolist(), keep.tolist(), first, recent, out.shape[3]))


def cache_compact(tensors, block_table, kept):
    for t, new in zip(tensors, plain_compact(tensors, block_table, kept)):
        t.copy_(new)


def token_logprobs(logits, ids, logprobs, entropy, top_ids=None, top_logprobs=None):
    lp, ent, ti, tl = plain_logprobs(logits, ids, 0 if top_ids is None else top_ids.shape[1])
    logprobs.copy_(lp), entropy.copy_(ent)
    if top_ids is not None:
        top_ids.copy_(ti), top_logprobs.copy_(tl)


STAND_INS = (attention_mass, evict_select, cache_compact, token_logprobs)


# -------------------------------------------------------------------------- a whole model with a bounded cache, in 64 bits
class PlainBounded:
    """One request of a Qwen2 model, its cache as lists of (position, key, value, sum) a layer and kv head, nothing paged."""

    def __init__(self, cfg, w):
        import plain_impl
        self.p, self.cfg, self.w = plain_impl, cfg, w
        self.nh, self.nkv, self.dh = cfg["num_attention_heads"], cfg["num_key_value_heads"], plain_impl.head_dim_of(cfg)
        heads = [[None] * self.nkv for _ in range(cfg["num_hidden_layers"])]
        self.k = [[np.zeros((0, self.dh))] * self.nkv for _ in heads]
        self.v = [[np.zeros((0, self.dh))] * self.nkv for _ in heads]
        self.mass = [[np.zeros(0)] * self.nkv for _ in heads]
        self.pos = 0

    @property
    def cached(self):
        return len(self.mass[0][0])

    def step(self, ids):
        p, cfg, w, nh, nkv, dh = self.p, self.cfg, self.w, self.nh, self.nkv, self.dh
        t, eps, theta = len(ids), cfg.get("rms_norm_eps", 1e-6), cfg.get("rope_theta", 10000.0)
        pos = np.arange(self.pos, self.pos + t)
        x = p.embedding(np.asarray(ids), w["model.embed_tokens.weight"])
        for l in range(cfg["num_hidden_layers"]):
            a = f"model.layers.{l}.self_attn."
            xn = p.rms_norm(x, w[f"model.layers.{l}.input_layernorm.weight"], eps)
            q, k, v = (p.linear(xn, w[a + f"{n}_proj.weight"], w.get(a + f"{n}_proj.bias")) for n in "qkv")
            q, k, v = p.rope_neox(q.reshape(t, nh, dh), pos, theta), p.rope_neox(k.reshape(t, nkv, dh), pos, theta), v.reshape(t, nkv, dh)
            out = np.zeros((t, nh, dh))
            for g in range(nkv):
                before = len(self.mass[l][g])
                self.k[l][g], self.v[l][g] = np.concatenate([self.k[l][g], k[:, g]]), np.concatenate([self.v[l][g], v[:, g]])
                self.mass[l][g] = np.concatenate([self.mass[l][g], np.zeros(t)])
                seen = np.arange(before + t)[None, :] <= before + np.arange(t)[:, None]
                for h in range(g * nh // nkv, (g + 1) * nh // nkv):
                    s = np.where(seen, q[:, h] @ self.k[l][g].T / math.sqrt(dh), -np.inf)
                    e = np.exp(s - s.max(1, keepdims=True))
                    e /= e.sum(1, keepdims=True)
                    out[:, h] = e @ self.v[l][g]
                    self.mass[l][g] = self.mass[l][g] + e.sum(0)
            x = x + p.linear(out.reshape(t, nh * dh), w[a + "o_proj.weight"])
            xn = p.rms_norm(x, w[f"model.layers.{l}.post_attention_layernorm.weight"], eps)
            m = f"model.layers.{l}.mlp."
            x = x + p.linear(p.swiglu(p.linear(xn, w[m + "gate_proj.weight"]), p.linear(xn, w[m + "up_proj.weight"])), w[m + "down_proj.weight"])
        self.pos += t
        head = w["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings") or "lm_head.weight" not in w else w["lm_head.weight"]
        return p.linear(p.rms_norm(x, w["model.norm.weight"], eps), head)

    def evict(self, keep, first=4, recent=None):
        recent = keep // 2 if recent is None else recent
        for l in range(len(self.mass)):
            for g in range(self.nkv):
                n, m = len(self.mass[l][g]), self.mass[l][g]
                if n <= keep:
                    continue
                last = min(recent, keep)
                front = min(first, keep - last)
                middle = np.arange(front, n - last)
                chosen = middle[np.argsort(-m[middle], kind="stable")][:keep - front - last]
                at = np.sort(np.concatenate([np.arange(front), chosen, np.arange(n - last, n)])).astype(int)
                self.k[l][g], self.v[l][g], self.mass[l][g] = self.k[l][g][at], self.v[l][g][at], m[at]


def bounded_run(eng, plain, tokens, portions, budget, slack, first, recent, others=(), rel=2e-5):
    """A text in portions (numbers of tokens) through the engine, cut to `budget` when it has outgrown the slack, beside requests
    `others` [(name, portions)] that are cut the same way; the logits of every token against the plain model's."""
    from litinfer_amd.engine import StepEntry
    names = {"text": (tokens, list(portions), plain("text"))}
    names.update({name: (toks, list(parts), plain(name)) for name, toks, parts in others})
    at = dict.fromkeys(names, 0)
    cuts = 0
    while any(parts for _, parts, _ in names.values()):
        entries, want = [], []
        for name, (toks, parts, ref) in names.items():
            if parts:
                n = parts.pop(0)
                chunk = toks[at[name]:at[name] + n]
                at[name] += n
                entries.append(StepEntry(name, chunk, list(range(len(chunk)))))
                want.append(ref.step(chunk))
        got = eng.step(entries).cpu().double().numpy()
        want = np.concatenate(want)
        assert np.abs(got - want).max() <= rel * np.abs(want).max(), float(np.abs(got - want).max() / np.abs(want).max())
        long = [e.rid for e in entries if eng.cache.cached_len(e.rid) > budget + slack]
        left = eng.evict(long, budget, first, recent) if long else []
        assert left == [budget] * len(long)
        for rid in long:
            names[rid][2].evict(budget, first, recent)
            cuts += 1
        for e in entries:
            assert eng.cache.cached_len(e.rid) == names[e.rid][2].cached
            assert eng.cache.table_len(e.rid, 0) >= -(-eng.cache.cached_len(e.rid) // eng.page_size)
        eng.cache.check_invariants()
    for name in names:
        eng.finish(name)
    assert eng.cache.free_pages() == [g.pool.capacity for g in eng.cache.groups]
    return cuts
