"""attention_mass held closely to its plain form in 64 bits, and keys that are not finite around the borders of what is seen.

The tolerance adds roundings as independent errors do: a rounding of a number of size x is off by at most 2^-24 x, 2^-24 x / sqrt(3) in the root
mean square; n of them by sqrt(n) times that, and six times that is not passed by any of some million numbers."""
import math

import pytest
import torch

import bounded_cache_cases as cases
from litinfer_amd.kernels import ops
from test_bounded_cache_gpu import mass_inputs, mass_tolerance

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24
DEV = "cuda:0"


def largest(qkv, k, meta, nh, nkv, dh, page_size, scale):
    """The largest partial sum of 16, 32, .. products of any score, and the largest log of a row's sum."""
    part, lse = 0.0, 0.0
    for r in range(meta.num_segments):
        q, c, at = int(meta.host_q_len[r]), int(meta.host_ctx_len[r]), int(meta.host_q_start[r])
        t = torch.arange(c, device=DEV)
        seen, page = t[None, :] <= torch.arange(c - q, c, device=DEV)[:, None], meta.block_table[r].long()[t // page_size]
        for h in range(nh):
            keys, rows = k[page, h * nkv // nh, t % page_size].double(), qkv[at:at + q, h * dh:(h + 1) * dh].double()
            s = torch.zeros(q, c, dtype=torch.float64, device=DEV)
            for d in range(0, dh, 16):
                s += rows[:, d:d + 16].contiguous() @ keys[:, d:d + 16].t().contiguous() * scale
                part = max(part, float(s.abs().max()))
            lse = max(lse, float(torch.logsumexp(s.masked_fill(~seen, -math.inf), 1).abs().max()))
    return part, lse


def close_tolerance(qkv, k, meta, nh, nkv, dh, page_size, scale):
    """Relative to a key's sum.  A weight's error is that of its score and of its row's log-sum (which is no more off than a score): dh + 4 roundings of
    partial sums each; the scale's own two; the difference, the log-sum as it is kept and its two parts, of their size; two exp2 and a log2 of two
    halves each.  The row's sum has at most half the keys in one chain, a key's sum a 32nd of its queries and heads (a quarter where the head size takes the
    plain kernels), and the joins' 32."""
    part, lse = largest(qkv, k, meta, nh, nkv, dh, page_size, scale)
    pairs, tiled = meta.max_q_len * (nh // nkv), dh * qkv.element_size() % 16 == 0

    def roots(n):
        return 6 * HALF * math.sqrt(n / 3)
    return (2 * roots(dh + 4) * part + 4 * HALF * part + 4 * HALF * max(part, lse) / math.log(2) + 8 * HALF
            + roots(meta.max_ctx_len / 2 + 32) + roots(pairs / (32 if tiled else 4) + 32))


def drawn_by(r, i, h, qkv, k, meta, nh, nkv, dh, page_size, scale):
    """The weights of query i of request r in head h (on the CPU)."""
    qkv, k, table = qkv.cpu().double(), k.cpu().double(), meta.block_table.cpu().long()
    q, c, at = int(meta.host_q_len[r]), int(meta.host_ctx_len[r]), int(meta.host_q_start[r])
    t = torch.arange(c - q + i + 1)
    return torch.softmax(k[table[r, t // page_size], h * nkv // nh, t % page_size] @ qkv[at + i, h * dh:(h + 1) * dh] * scale, 0)


def in_ten_bits(w):
    m, e = torch.frexp(w)
    return torch.ldexp(torch.round(m * 1024) / 1024, e)


BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("segs,nh,nkv,dh,dtype", [
    ([(910, 3410), (1, 33), (70, 75)], 64, 64, 64, BF),              # two tiles of keys a wave
    ([(910, 6333)], 32, 32, 128, BF),
    ([(910, 10800)], 17, 17, 256, BF),
    ([(517, 1311), (1, 700)], 12, 12, 128, BF),                      # one tile
    ([(517, 1311), (1, 700)], 12, 12, 128, F32),
    ([(910, 2000)], 8, 4, 64, F32),
    ([(300, 900)], 3, 3, 256, F32),
    ([(129, 300), (1, 70)], 4, 4, 36, BF),                           # no whole pieces: the plain kernels
    ([(129, 300), (1, 70)], 4, 2, 33 * 2, F32),
    ([(1, 5001), (1, 3), (1, 2500), (1, 640)], 12, 12, 128, BF),     # single tokens, scores in memory
    ([(1, 5001), (1, 3), (1, 2500), (1, 640)], 12, 12, 128, F32),
    ([(1, 400), (1, 3), (1, 65)], 12, 12, 128, BF),                  # in one kernel
    ([(1, 400), (1, 3), (1, 65)], 12, 12, 64, F32)])
def test_mass_is_as_close_as_its_roundings_allow(segs, nh, nkv, dh, dtype):
    page_size, scale = 16, 1.0 / math.sqrt(dh)
    qkv, mass, k, meta = mass_inputs(segs, nh, nkv, dh, page_size, dtype)
    mass.zero_()
    args = (qkv, k, meta, nh, nkv, dh, page_size, scale)
    want = cases.plain_mass(qkv, mass, k, meta, nh, nkv, dh, page_size, scale)
    tol = close_tolerance(*args)
    assert tol < 2e-4
    ops.attention_mass(qkv, mass, k, meta, nh, nkv, dh, page_size, scale)
    got = mass.cpu().double()
    off = ((got - want).abs() / want.clamp(min=1e-300)).masked_fill(want == 0, 0.0)
    print(f"off by {float(off.max()):.2e}, tolerance {tol:.2e}")
    assert bool((got[want == 0] == 0).all()) and float(off.max()) <= tol
    # what the tolerance is worth: one query of one head too few, and weights of 10 bits, would be seen
    q, c = segs[0]
    t = torch.arange(c)
    page = meta.block_table.cpu().long()[0, t // page_size]
    for g in (0, nkv - 1):
        sums, heads, last = want[page, g, t % page_size, 0], range(g * nh // nkv, (g + 1) * nh // nkv), min(q, 16)
        if q > 1:
            lost = drawn_by(0, q // 2, heads[0], *args)
            assert float((lost / sums[:len(lost)] > tol).double().mean()) > 0.5
        # (the last keys, which few queries see; a single query's all)
        rough = sum(torch.nn.functional.pad(in_ten_bits(w), (0, c - len(w))) for w in (drawn_by(0, i, h, *args) for i in range(q - last, q) for h in heads))
        seen = slice(c - last if q > 1 else 0, c)
        assert float(((rough - sums).abs() / sums)[seen].max()) > tol


# ----------------------------------------------------------------------------------------------- not finite
# one tile a wave; two; the plain kernels
SHAPES = [([(70, 200), (33, 33), (1, 40), (129, 300), (1, 1000)], 4, 2, 64, BF), ([(70, 200), (33, 33), (1, 40), (129, 300), (1, 1000)], 4, 2, 64, F32),
          ([(910, 3410), (70, 75), (1, 40), (33, 33)], 64, 8, 64, BF), ([(70, 200), (33, 33), (1, 40)], 4, 2, 36, BF), ([(65, 200), (1, 40), (20, 20)], 6, 1, 256, BF)]


def with_a_page_of_nobody(segs, nh, nkv, dh, dtype, holes=()):
    """The batch with page 0 in nobody's table, and which rows of the pool a request holds."""
    qkv, mass, k, meta = mass_inputs(segs, nh, nkv, dh, 16, dtype, holes=holes)
    k, mass = torch.cat([torch.zeros_like(k[:1]), k]), torch.cat([torch.ones_like(mass[:1]), mass])
    meta.block_table = torch.where(meta.block_table >= 0, meta.block_table + 1, -1).to(torch.int32)
    held = torch.zeros(mass.shape, dtype=torch.bool, device=DEV)
    for r, c in enumerate(meta.host_ctx_len.tolist()):
        t = torch.arange(c, device=DEV)
        page = meta.block_table[r].long()[t // 16]
        held[page[page >= 0], :, (t % 16)[page >= 0]] = True
    return qkv, mass, k, meta, held


@pytest.mark.parametrize("segs,nh,nkv,dh,dtype", SHAPES)
@pytest.mark.parametrize("holes", [(), ((0, 2), (0, 7), (2, 0), (1, 1))])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_lies_in_rows_that_nobody_sees_changes_nothing(segs, nh, nkv, dh, dtype, holes, value):
    """Behind the last token in its page, in pages of nobody, and in page 0, whose rows stand in for those of pages that are not there."""
    qkv, mass, k, meta, held = with_a_page_of_nobody(segs, nh, nkv, dh, dtype, holes)
    scale, out = dh ** -0.5, []
    assert not held[0].any() and (~held).sum() > 8 * nkv
    for x in (0.0, value):
        now = mass.clone()
        ops.attention_mass(qkv, now, torch.where(held, k, torch.full_like(k, x)), meta, nh, nkv, dh, 16, scale)
        out.append(now)
    assert torch.equal(out[0], out[1]) and torch.isfinite(out[0]).all() and torch.equal(out[0][~held], mass[~held])


@pytest.mark.parametrize("segs,nh,nkv,dh,dtype", SHAPES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_key_that_is_not_finite_leaves_its_own_request_and_head_without_sums_and_nobody_else(segs, nh, nkv, dh, dtype, value):
    """At a place of the portion that only its last queries see, and that others' tiles hold too."""
    qkv, mass, k, meta, held = with_a_page_of_nobody(segs, nh, nkv, dh, dtype)
    scale, clean = dh ** -0.5, mass.clone()
    ops.attention_mass(qkv, clean, k, meta, nh, nkv, dh, 16, scale)
    for r, back in ((0, 1), (0, 40), (1, 2)):
        place = segs[r][1] - back
        bad, now = k.clone(), mass.clone()
        bad[int(meta.block_table[r, place // 16]), nkv - 1, place % 16] = value
        ops.attention_mass(qkv, now, bad, meta, nh, nkv, dh, 16, scale)
        t = torch.arange(segs[r][1], device=DEV)
        mine = torch.zeros_like(held)
        mine[meta.block_table[r].long()[t // 16], nkv - 1, t % 16] = True
        assert torch.isnan(now[mine]).all() and torch.equal(now[~mine], clean[~mine])


@pytest.mark.parametrize("segs,nh,nkv,dh,dtype", SHAPES)
def test_keys_whose_scores_are_minus_infinity_draw_nothing(segs, nh, nkv, dh, dtype):
    """At the borders of tiles and of the portion, cached ones and new ones."""
    qkv, mass, k, meta, held = with_a_page_of_nobody(segs, nh, nkv, dh, dtype)
    scale = dh ** -0.5
    qkv[:, 0:nh * dh:dh] = qkv[:, 0:nh * dh:dh].abs() + 0.5          # (the first element of every query's head)
    tol = mass_tolerance(qkv, k, meta, nh, nkv, dh, scale)
    nothing = torch.zeros_like(held)
    for r, (q, c) in enumerate(segs):
        for place in {1, 31, 32, 63, 64, c - q - 1, c - q, c - q + 1, c - 2}:
            if 0 < place < c and not (q == 1 and place == c - 1):
                page = int(meta.block_table[r, place // 16])
                k[page, :, place % 16] = 0.0
                k[page, :, place % 16, 0] = -math.inf
                nothing[page, :, place % 16] = True
    want = cases.plain_mass(qkv, mass, k, meta, nh, nkv, dh, 16, scale)
    before = mass.clone()
    ops.attention_mass(qkv, mass, k, meta, nh, nkv, dh, 16, scale)
    got = mass.cpu().double()
    assert torch.isfinite(got).all() and bool(((got - want).abs() <= tol * want.abs() + 1e-30).all())
    assert bool(((mass == before) | (mass == 0.0))[nothing].all())


@pytest.mark.parametrize("segs,nh,nkv,dh,dtype", SHAPES)
def test_rows_all_of_whose_scores_are_minus_infinity_add_nothing(segs, nh, nkv, dh, dtype):
    """One kv head's keys throughout, of portions and single tokens: its cached keys keep their sums, its new ones have none."""
    qkv, mass, k, meta, held = with_a_page_of_nobody(segs, nh, nkv, dh, dtype)
    qkv[:, 0:nh * dh:dh] = qkv[:, 0:nh * dh:dh].abs() + 0.5
    scale, clean, start = dh ** -0.5, mass.clone(), mass.clone()
    ops.attention_mass(qkv, clean, k, meta, nh, nkv, dh, 16, scale)
    k[:, nkv - 1] = 0.0
    k[:, nkv - 1, :, 0] = -math.inf
    ops.attention_mass(qkv, mass, k, meta, nh, nkv, dh, 16, scale)
    assert torch.equal(mass[:, :nkv - 1], clean[:, :nkv - 1])
    fresh = torch.zeros_like(held)
    for r, (q, c) in enumerate(segs):
        t = torch.arange(c - q, c, device=DEV)
        fresh[meta.block_table[r].long()[t // 16], :, t % 16] = True
    assert torch.equal(mass[:, nkv - 1], start.masked_fill(fresh, 0.0)[:, nkv - 1])
