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
