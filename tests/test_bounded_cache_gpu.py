"""The operators around a cache of bounded length, and token_logprobs, against their plain forms in 64 bits.

Tolerances are worked out from the arithmetic: float32 rounds by at most 2^-24 relative to the value."""
import math

import pytest
import torch

import bounded_cache_cases as cases
from litinfer_amd.engine.workspace import Workspace
from litinfer_amd.kernels import ops

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24
DEV = "cuda:0"


# ------------------------------------------------------------------------------------------------ attention_mass
def mass_inputs(segs, nh, nkv, dh, page_size, dtype, seed=0, extra_columns=0, holes=(), width=1.5):
    meta, pages = cases.batch(segs, page_size, DEV, seed, holes=holes)
    g = torch.Generator().manual_seed(seed + 1)
    qkv = (torch.randn(meta.num_tokens, (nh + 2 * nkv) * dh + extra_columns, generator=g) * width).to(dtype).to(DEV)
    k = torch.randn(pages, nkv, page_size, dh, generator=g).to(dtype).to(DEV)
    mass = (torch.rand(pages, nkv, page_size, 1, generator=g)).to(DEV)
    return qkv, mass, k, meta


def mass_tolerance(qkv, k, meta, nh, nkv, dh, scale):
    """Relative: a score is off by (dh + 4) roundings of the sum of its products' sizes, the log of a row's sum by the same and a rounding a
    key, exp2 and log2 by 2^-22, a key's sum by a rounding a query and head."""
    rows = qkv[:, :nh * dh].float().abs().view(-1, nh, dh).amax((0, 1)).cpu()
    keys = k.float().abs().nan_to_num().amax((0, 1, 2)).cpu()
    size = min(float((rows * keys).sum()), float(qkv[:, :nh * dh].float().view(-1, nh, dh).norm(dim=-1).max() * k.float().nan_to_num().norm(dim=-1).max())) * scale
    return 2 * (dh + 4) * HALF * size + (meta.max_ctx_len + meta.max_q_len * (nh // nkv) + 16) * HALF


def check_mass(segs, nh, nkv, dh, page_size, dtype, fresh=True, seed=0, holes=(), extra_columns=0, ws=None, scale=None):
    qkv, mass, k, meta = mass_inputs(segs, nh, nkv, dh, page_size, dtype, seed, extra_columns, holes)
    scale = 1.0 / math.sqrt(dh) if scale is None else scale
    want = cases.plain_mass(qkv, mass, k, meta, nh, nkv, dh, page_size, scale, fresh)
    ops.attention_mass(qkv, mass, k, meta, nh, nkv, dh, page_size, scale, fresh=fresh, ws=ws)
    got = mass.cpu().double()
    tol = mass_tolerance(qkv, k, meta, nh, nkv, dh, scale)
    assert torch.isfinite(got).all()
    off = (got - want).abs() - tol * want.abs() - 1e-30
    assert float(off.max()) <= 0, (float(((got - want).abs() / want.abs().clamp(min=1e-30)).max()), tol)


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,dh,page_size", [(14, 2, 64, 16), (12, 2, 128, 16), (28, 4, 128, 8), (4, 4, 128, 16), (40, 2, 64, 32), (6, 1, 256, 16),
                                                 (5, 5, 80, 5), (4, 2, 36, 3), (3, 1, 2, 1), (33, 1, 96, 16)])
def test_mass_of_single_tokens(dtype, nh, nkv, dh, page_size):
    check_mass([(1, 1), (1, 2), (1, 16), (1, 17), (1, 333), (1, 64), (1, 65)], nh, nkv, dh, page_size, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,dh,page_size", [(14, 2, 64, 16), (12, 2, 128, 16), (28, 4, 128, 7), (6, 1, 256, 16), (5, 5, 80, 5), (4, 2, 36, 3), (17, 1, 8, 4)])
def test_mass_of_portions_beside_single_tokens(dtype, nh, nkv, dh, page_size):
    check_mass([(2, 2), (1, 40), (33, 33), (129, 300), (1, 1), (64, 64), (65, 130), (3, 200)], nh, nkv, dh, page_size, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_mass_of_a_long_portion_and_long_contexts(dtype):
    check_mass([(517, 1311)], 12, 2, 128, 16, dtype)
    check_mass([(1, 5001), (1, 3)], 28, 4, 128, 16, dtype, ws=Workspace(DEV))
    check_mass([(700, 700), (1, 2049), (300, 900)], 14, 2, 64, 16, dtype, ws=Workspace(DEV))


@pytest.mark.parametrize("nh,nkv,dh,ctx,holes", [(64, 2, 64, 3410, []), (64, 8, 80, 3411, [(0, 3), (0, 40), (0, 213)]), (32, 2, 128, 6333, []), (17, 1, 256, 10800, [(0, 0)])])
def test_mass_of_portions_with_work_for_many_rounds(nh, nkv, dh, ctx, holes):
    """So many pairs of a head and a stage of queries that a wave takes two tiles of keys."""
    check_mass([(910, ctx), (1, 33), (70, 75)], nh, nkv, dh, 16, torch.bfloat16, holes=holes)


@pytest.mark.parametrize("dtype", DTYPES)
def test_mass_that_adds_to_keys_of_another_entry(dtype):
    check_mass([(1, 70), (40, 90), (2, 2)], 12, 2, 128, 16, dtype, fresh=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_mass_with_wider_rows_another_scale_and_pages_that_are_not_there(dtype):
    check_mass([(1, 70), (40, 90)], 12, 2, 128, 16, dtype, extra_columns=3)
    check_mass([(1, 70), (40, 90)], 12, 2, 64, 16, dtype, scale=0.9)
    # (the one query of request 2 sees nothing at all)
    check_mass([(1, 170), (40, 290), (1, 16), (7, 20)], 4, 2, 64, 16, dtype, holes=[(0, 2), (0, 3), (1, 0), (1, 9), (2, 0), (3, 0)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_mass_leaves_what_no_request_holds_and_makes_the_same_bits_twice(dtype):
    qkv, mass, k, meta = mass_inputs([(1, 130), (90, 200), (1, 33)], 12, 2, 128, 16, dtype)
    before = mass.clone()
    again = mass.clone()
    scale = 128 ** -0.5
    ops.attention_mass(qkv, mass, k, meta, 12, 2, 128, 16, scale)
    ops.attention_mass(qkv, again, k, meta, 12, 2, 128, 16, scale)
    assert torch.equal(mass, again)
    held = torch.zeros_like(mass, dtype=torch.bool)
    for r, c in enumerate(meta.host_ctx_len.tolist()):
        t = torch.arange(c, device=DEV)
        held[meta.block_table[r].long()[t // 16], :, t % 16] = True
    assert torch.equal(mass[~held], before[~held])
    # every query and head gives one unit in all: the fresh keys' sums and what the others have more than before
    fresh = torch.zeros_like(held)
    for r, (q, c) in enumerate(zip(meta.host_q_len.tolist(), meta.host_ctx_len.tolist())):
        t = torch.arange(c - q, c, device=DEV)
        fresh[meta.block_table[r].long()[t // 16], :, t % 16] = True
    total = float((mass.double() - before.double().masked_fill(fresh, 0.0))[held].sum())
    # (each sum is off by what the scores allow, and by a rounding of what was there before)
    allowed = mass_tolerance(qkv, k, meta, 12, 2, 128, scale) * 92 * 12 + HALF * float(before.sum())
    assert abs(total - 92 * 12) <= allowed


@pytest.mark.parametrize("dtype", DTYPES)
def test_mass_of_infinite_and_undefined_keys(dtype):
    """A key so far behind that its weight is nothing, and a NaN key: who sees it has no weights, others are untouched."""
    qkv, mass, k, meta = mass_inputs([(1, 50), (1, 40)], 4, 2, 64, 16, dtype)
    page = int(meta.block_table[0, 1])
    k[page, 0, 3] = math.nan
    ops.attention_mass(qkv, mass, k, meta, 4, 2, 64, 16, 0.125)
    t = torch.arange(50, device=DEV)
    first = mass[meta.block_table[0].long()[t // 16], :, t % 16, 0]
    assert torch.isnan(first[:, 0]).all() and torch.isfinite(first[:, 1]).all()
    t = torch.arange(40, device=DEV)
    assert torch.isfinite(mass[meta.block_table[1].long()[t // 16], :, t % 16, 0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_mass_of_many_requests(dtype):
    """More than a launch names one by one: single tokens alone, portions alone, both."""
    check_mass([(1, 3 + 5 * i) for i in range(70)], 4, 2, 64, 16, dtype)
    check_mass([(2 + i % 3, 9 + 3 * i) for i in range(70)], 4, 2, 64, 16, dtype)
    check_mass([(1 if i % 2 else 2 + i % 5, 9 + 3 * i) for i in range(150)], 4, 2, 64, 16, dtype)
    check_mass([(1, 600)] * 130, 4, 2, 64, 16, dtype)


def test_operators_on_the_last_pages_of_a_large_pool():
    """Keys whose place in the pool passes 2^31 elements, and 2^32 bytes."""
    pages, nkv, dh = 300000, 4, 128
    k = torch.zeros(1, pages, nkv, 16, dh, dtype=torch.bfloat16, device=DEV)
    mass = torch.zeros(1, pages, nkv, 16, 1, device=DEV)
    small, _ = cases.batch([(1, 400), (70, 300), (1, 30)], 16, DEV, 3)
    g = torch.Generator().manual_seed(9)
    used = int(small.block_table.max()) + 1
    few_k, few_mass = torch.randn(1, used, nkv, 16, dh, generator=g).bfloat16().to(DEV), torch.rand(1, used, nkv, 16, 1, generator=g).to(DEV)
    k[:, pages - used:], mass[:, pages - used:] = few_k, few_mass
    qkv = torch.randn(72, 12 * dh + 2 * nkv * dh, generator=g).bfloat16().to(DEV)
    far, _ = cases.batch([(1, 400), (70, 300), (1, 30)], 16, DEV, 3)
    far.block_table = torch.where(far.block_table >= 0, far.block_table + (pages - used), -1).to(torch.int32)
    lens, keep = ints([400, 300, 30]), ints([100, 90, 20])
    out = []
    for pool_k, pool_m, meta in ((few_k, few_mass, small), (k, mass, far)):
        ops.attention_mass(qkv, pool_m[0], pool_k[0], meta, 12, nkv, dh, 16, dh ** -0.5)
        kept = torch.empty(1, 3, nkv, 100, dtype=torch.int32, device=DEV)
        ops.evict_select(pool_m, meta.block_table, lens, keep, 4, 20, kept)
        ops.cache_compact([pool_k, pool_m], meta.block_table, kept)
        out.append((kept, pool_k[:, -used:].clone(), pool_m[:, -used:].clone()))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert not k[:, :pages - used].any() and not mass[:, :pages - used].any()


def test_mass_of_a_batch_that_has_changed_since():
    """What is looked at once a step is looked at again for other arrays, and a batch that has grown in place is refused."""
    qkv, mass, k, meta = mass_inputs([(1, 50), (1, 600)], 4, 2, 64, 16, torch.bfloat16)
    args = (4, 2, 64, 16, 0.125)
    ops.attention_mass(qkv, mass, k, meta, *args)
    other = mass_inputs([(1, 40), (1, 500)], 4, 2, 64, 16, torch.bfloat16)[3]
    for name in ("q_start", "q_len", "ctx_len", "host_q_start", "host_q_len", "host_ctx_len"):
        setattr(meta, name, getattr(other, name))
    meta.max_ctx_len = other.max_ctx_len
    want = cases.plain_mass(qkv, mass, k, meta, *args)
    ops.attention_mass(qkv, mass, k, meta, *args)
    assert torch.allclose(mass.cpu().double(), want, rtol=mass_tolerance(qkv, k, meta, 4, 2, 64, 0.125), atol=1e-30)
    short = mass_inputs([(1, 5), (1, 600)], 4, 2, 64, 16, torch.bfloat16)
    meta = short[3]
    meta.block_table = torch.cat([meta.block_table, torch.full((2, 400), -1, dtype=torch.int32, device=DEV)], 1)
    meta.max_blocks = meta.block_table.shape[1]
    ops.attention_mass(short[0], short[1], short[2], meta, *args)
    meta.host_ctx_len[0] = 6000
    with pytest.raises(RuntimeError, match="refused"):
        ops.attention_mass(short[0], short[1], short[2], meta, *args)


def test_mass_in_a_recording_and_on_another_stream():
    qkv, mass, k, meta = mass_inputs([(1, 130), (1, 260), (1, 33)], 12, 2, 128, 16, torch.bfloat16)
    want = mass.clone()
    ws = Workspace(DEV)
    args = (k, meta, 12, 2, 128, 16, 128 ** -0.5)
    ops.attention_mass(qkv, want, *args, ws=ws)
    start, side = mass.clone(), torch.cuda.Stream()
    meta.padded = True
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        ops.attention_mass(qkv, mass, *args, ws=ws)
    for _ in range(3):
        mass.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mass, want)
        torch.randn(1000, device=DEV).sum().item()
    # longer contexts of the same tables in a replay
    meta.ctx_len.add_(7)
    mass.copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    meta.host_ctx_len = meta.host_ctx_len + 7
    plain = cases.plain_mass(qkv, start, k, meta, 12, 2, 128, 16, 128 ** -0.5)
    assert torch.allclose(mass.cpu().double(), plain, rtol=mass_tolerance(qkv, k, meta, 12, 2, 128, 128 ** -0.5), atol=1e-30)


@pytest.mark.parametrize("segs", [[(1, 30), (1, 31)], [(1, 700), (1, 90)]])
def test_mass_of_a_replay_that_is_told_more_than_the_tables_hold(segs):
    """Lengths are cut to the tables: nothing behind them is read or written."""
    qkv, mass, k, meta = mass_inputs(segs, 4, 2, 64, 5, torch.bfloat16)
    meta.padded = True
    args = (4, 2, 64, 5, 0.125)
    room = meta.max_blocks * 5
    start = mass.clone()
    meta.ctx_len.fill_(room)
    ops.attention_mass(qkv, mass, k, meta, *args)
    want = mass.clone()
    mass.copy_(start)
    meta.ctx_len.fill_(room + 1000)
    ops.attention_mass(qkv, mass, k, meta, *args)
    assert torch.equal(mass, want) and torch.isfinite(mass).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_mass_of_portions_in_a_recording(dtype):
    qkv, mass, k, meta = mass_inputs([(1, 130), (97, 260), (1, 33), (300, 300)], 12, 2, 128, 16, dtype)
    args = (k, meta, 12, 2, 128, 16, 128 ** -0.5)
    start, ws = mass.clone(), Workspace(DEV)
    ops.attention_mass(qkv, mass, *args, ws=ws)
    want = mass.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_mass(qkv, mass, *args, ws=ws)
    for _ in range(3):
        mass.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mass, want)
        torch.randn(100000, device=DEV).sum().item()


# ------------------------------------------------------------------------------------- evict_select, cache_compact
def cache(lens, entries, nkv, page_size, seed=0, holes=()):
    meta, pages = cases.batch([(1, max(n, 1)) for n in lens], page_size, DEV, seed, holes=holes)
    g = torch.Generator().manual_seed(seed + 5)
    mass = torch.exp(2 * torch.randn(entries, pages, nkv, page_size, 1, generator=g))
    return meta.block_table, mass.to(DEV), pages, g


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check_select(mass, table, lens, keep, first, recent, room):
    entries, _, nkv, _, _ = mass.shape
    out = torch.full((entries, len(lens), nkv, room), 12345, dtype=torch.int32, device=DEV)
    ops.evict_select(mass, table, ints(lens), ints(keep), first, recent, out)
    want = cases.plain_select(mass, table, lens, keep, first, recent, room)
    assert torch.equal(out.cpu(), want)
    return out


@pytest.mark.parametrize("page_size", [16, 1, 7])
@pytest.mark.parametrize("first,recent", [(0, 0), (4, 8), (0, 300), (300, 0), (5, 11)])
def test_select(page_size, first, recent):
    lens = [0, 1, 2, 15, 16, 17, 40, 255, 256, 257, 700]
    keep = [4, 1, 1, 15, 3, 20, 0, 16, 255, 100, 300]
    table, mass, _, _ = cache(lens, 3, 2, page_size)
    check_select(mass, table, lens, keep, first, recent, 300)
    check_select(mass, table, lens, keep, first, recent, 17)          # less room than was asked for


def test_select_of_equal_sums_zeros_infinities_and_undefined_ones():
    lens, keep = [300, 300, 300, 40], [100, 37, 290, 20]
    table, mass, _, g = cache(lens, 2, 3, 16, holes=[(1, 4), (2, 0)])
    mass[0] = 1.5                                                     # all equal: the lowest places
    mass[1] = torch.randint(0, 3, mass[1].shape, generator=g).float().to(DEV)
    flat = mass[1].view(-1)
    flat[::7], flat[1::11], flat[2::13], flat[3::17], flat[4::19] = math.nan, math.inf, -math.inf, -0.0, -1.0
    for first, recent in ((0, 0), (4, 16)):
        check_select(mass, table, lens, keep, first, recent, 290)


def test_select_of_long_requests():
    lens, keep = [9001, 40000, 33000], [2000, 30001, 64]
    table, mass, _, g = cache(lens, 1, 2, 16)
    mass[torch.rand(mass.shape, generator=g).to(DEV) < 0.3] = 0.0
    check_select(mass, table, lens, keep, 4, 50, 30001)


@pytest.mark.parametrize("longest", [1023, 1025, 4000, 4097, 16000, 16400, 32000, 33000])
def test_select_of_every_length(longest):
    """Each form of the kernel, with sums that are all different and sums of which many are equal."""
    lens, keep = [longest, longest // 2, 3], [longest // 3, 5, 3]
    table, mass, _, g = cache(lens, 1, 1, 16)
    check_select(mass, table, lens, keep, 2, 9, longest // 3)
    check_select(torch.floor(mass), table, lens, keep, 2, 9, longest // 3)


@pytest.mark.parametrize("longest", [300, 3000, 9000])
def test_select_of_sums_that_do_not_begin_on_16_bytes(longest):
    lens, keep = [longest, longest - 7, 30], [longest // 2, 9, 30]
    table, mass, _, _ = cache(lens, 2, 2, 16)
    for off in (1, 2, 3):
        view = torch.full((mass.numel() + off,), 1e9, device=DEV)[off:].view(mass.shape)
        view.copy_(mass)
        check_select(view, table, lens, keep, 3, 10, longest // 2)


@pytest.mark.parametrize("page_size", [16, 5])
@pytest.mark.parametrize("shapes", [[(64, torch.bfloat16)] * 2 + [(1, torch.float32)], [(128, torch.float32)] * 2 + [(1, torch.float32)],
                                    [(36, torch.bfloat16), (2, torch.bfloat16)], [(256, torch.bfloat16)], [(3, torch.float32), (6, torch.bfloat16)] * 2])
def test_compact(page_size, shapes):
    lens, keep = [1, 2, 33, 700, 256, 513], [1, 1, 30, 333, 256, 16]
    table, mass, pages, g = cache(lens, 2, 3, page_size)
    kept = check_select(mass, table, lens, keep, 4, 10, 333)
    tensors = [torch.randn(2, pages, 3, page_size, d, generator=g).to(dt).to(DEV) for d, dt in shapes]
    want = cases.plain_compact(tensors, table, kept)
    ops.cache_compact(tensors, table, kept)
    for a, b in zip(tensors, want):
        assert torch.equal(a.cpu(), b)


def test_compact_of_a_long_request_and_of_places_that_are_not_there():
    lens, keep = [9001, 12], [4001, 12]
    table, mass, pages, g = cache(lens, 1, 2, 16)
    kept = check_select(mass, table, lens, keep, 0, 0, 4001)
    k = torch.randn(1, pages, 2, 16, 128, generator=g).to(torch.bfloat16).to(DEV)
    want = cases.plain_compact([k], table, kept)
    ops.cache_compact([k], table, kept)
    assert torch.equal(k.cpu(), want[0])
    before = k.clone()
    kept.fill_(1 << 30)                                              # beyond the table
    ops.cache_compact([k], table, kept)
    kept.copy_(torch.arange(kept.shape[3], dtype=torch.int32, device=DEV) + 1)
    ops.cache_compact([k], torch.full_like(table, -1), kept)          # on pages that are not there
    ops.cache_compact([k], torch.full_like(table, pages), kept)
    assert torch.equal(k, before)


def test_select_and_compact_in_a_recording():
    lens, keep = [700, 90], [300, 64]
    table, mass, pages, g = cache(lens, 2, 2, 16)
    k = torch.randn(2, pages, 2, 16, 64, generator=g).to(torch.bfloat16).to(DEV)
    out = torch.empty(2, 2, 2, 300, dtype=torch.int32, device=DEV)
    n, m = ints(lens), ints(keep)
    start = [k.clone(), mass.clone()]
    ops.evict_select(mass, table, n, m, 4, 16, out)
    ops.cache_compact([k, mass], table, out)
    want = [k.clone(), mass.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.evict_select(mass, table, n, m, 4, 16, out)
        ops.cache_compact([k, mass], table, out)
    for _ in range(3):
        k.copy_(start[0]), mass.copy_(start[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, want[0]) and torch.equal(mass, want[1])
        torch.randn(1000, device=DEV).sum().item()


# ------------------------------------------------------------------------------------------------- token_logprobs
def logprob_call(x, ids, top):
    n = x.shape[0]
    lp, ent = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    ti, tl = (torch.empty(n, top, dtype=torch.int32, device=DEV), torch.empty(n, top, device=DEV)) if top else (None, None)
    ops.token_logprobs(x, ids, lp, ent, ti, tl)
    return lp, ent, ti, tl


def check_logprobs(x, ids, top):
    """A row's sum: at most 32 + 6 + 8 + 16 roundings of shares of one sign, each share off by 4 roundings and the rounding of its
    exponent (whose weight |d| exp(d) is below 0.37); the two differences one each."""
    lp, ent, ti, tl = logprob_call(x, ids, top)
    wlp, went, wti, wtl = cases.plain_logprobs(x, ids, top)

    def near(a, b, tol):
        a = a.cpu().double()
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        fine = torch.isfinite(b)
        assert bool(((a - b)[fine].abs() <= tol[fine]).all()), float((a - b)[fine].abs().max())
        assert torch.equal(a[torch.isinf(b)], b[torch.isinf(b)])
    near(lp, wlp, (80 + 3 * wlp.abs()) * HALF)
    near(ent, went, 160 * HALF * (1 + went))
    if top:
        assert torch.equal(ti.cpu(), wti)
        near(tl, wtl, (80 + 3 * wtl.abs()) * HALF)


@pytest.mark.parametrize("n,v,top", [(1, 1, 1), (1, 2, 2), (3, 5, 5), (2, 255, 20), (2, 256, 32), (1, 257, 32), (5, 1000, 3), (40, 3001, 32), (1, 151936, 20),
                                     (7, 152064, 5), (33, 32003, 0), (64, 50021, 1), (17, 8192, 8)])
def test_logprobs(n, v, top):
    g = torch.Generator().manual_seed(n * 1000 + v)
    x = (torch.randn(n, v, generator=g) * 3).to(DEV)
    check_logprobs(x, ints(torch.randint(0, v, (n,), generator=g).tolist()), top)
    x[:, :v // 2] = x[:, v - v // 2:]                                  # every logit twice: the lower id first
    check_logprobs(x, ints([v - 1] * n), top)


def test_logprobs_of_sure_rows_keep_their_digits():
    """One token far ahead: its log probability and the entropy are small sums of the others."""
    x = torch.zeros(4, 50000, device=DEV)
    x[0, 7], x[1, 49999], x[2, 300], x[3, 1] = 25.0, 40.0, 15.0, 30.0
    lp, ent, _, _ = logprob_call(x, ints([7, 49999, 300, 1]), 3)
    y = torch.log_softmax(x.cpu().double(), 1)
    p = torch.exp(y)
    r = (49999 * torch.exp(-torch.tensor([25.0, 40.0, 15.0, 30.0], dtype=torch.float64)))
    assert torch.allclose(lp.cpu().double(), -torch.log1p(r), rtol=80 * HALF, atol=0)
    d = torch.tensor([25.0, 40.0, 15.0, 30.0], dtype=torch.float64)
    assert torch.allclose(ent.cpu().double(), torch.log1p(r) + r * d / (1 + r), rtol=160 * HALF, atol=0)


def test_logprobs_of_masked_equal_and_undefined_rows():
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(9, 5003, generator=g) * 2).to(DEV)
    x[0, ::2] = -math.inf                                             # masked tokens
    x[1] = -math.inf
    x[1, 77] = 3.0                                                    # one token left
    x[2] = 1.25                                                       # all equal
    x[3] = -math.inf                                                  # nothing left
    x[4, 9] = math.inf
    x[5, 5000] = math.nan
    x[6] = torch.finfo(torch.float32).min                             # the type's lowest value throughout
    x[7, 100:] = torch.finfo(torch.float32).min
    x[8] = torch.sort(x[8], descending=True).values                   # the likeliest tokens side by side
    for ids in ([0] * 9, [1, 77, 5002, 4, 9, 5000, 2, 4000, 0], [-1, 5003, 1 << 30, -5, 9, 0, 0, 0, 1]):
        check_logprobs(x, ints(ids), 32)


def test_logprobs_of_rows_that_lie_apart_and_do_not_begin_on_16_bytes():
    g = torch.Generator().manual_seed(4)
    room = (torch.randn(6, 5011, generator=g) * 2).to(DEV)
    check_logprobs(room[:, 1:5000], ints([3] * 6), 7)
    check_logprobs(room[:, 3:4099], ints([4000] * 6), 7)
    check_logprobs(room[2:3, 2:], ints([0]), 32)


def test_logprobs_of_many_rows():
    x = torch.randn(70000, 40, device=DEV)
    check_logprobs(x, ints([39] * 70000), 2)


def test_logprobs_in_a_recording_beside_other_calls():
    x = torch.randn(5, 30011, device=DEV)
    ids = ints([1, 2, 3, 4, 5])
    lp, ent, ti, tl = logprob_call(x, ids, 4)
    out = [torch.empty_like(t) for t in (lp, ent, ti, tl)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.token_logprobs(x, ids, *out)
    big = torch.randn(100, 50000, device=DEV)
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        logprob_call(big, ints([0] * 100), 3)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, (lp, ent, ti, tl)))


def test_two_streams_at_once():
    x, y = torch.randn(64, 60000, device=DEV), torch.randn(64, 60000, device=DEV)
    ids = ints([5] * 64)
    want = [logprob_call(t, ids, 5) for t in (x, y)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        got = []
        for s, t in zip(streams, (x, y)):
            with torch.cuda.stream(s):
                got.append(logprob_call(t, ids, 5))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
