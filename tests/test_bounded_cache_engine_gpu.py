"""The engine with a cache of bounded length, its kernels and its recorded steps, against a whole model in 64 bits; log probabilities
through the scheduler and the entry point."""
import numpy as np
import pytest
import torch

import bounded_cache_cases as cases
import helpers
import plain_impl
from litinfer_amd.engine import Engine, Scheduler, StepEntry
from litinfer_amd.models import Qwen2
from tiny_configs import TINY_A, TINY_B, TINY_C, TINY_D, TINY_E

pytestmark = pytest.mark.gpu


def all_keys(cfg):
    return {**cfg, "use_sliding_window": False, "max_position_embeddings": 1024}


def text(n, vocab, seed=0):
    return np.random.default_rng(seed).integers(0, vocab, n).tolist()


def engine(d, dtype="float32", **kw):
    return Engine.from_dir(d, **{**dict(dtype=dtype, page_size=16, max_seqs=16, max_tokens=4000, attention_mass=True, page_order_seed=1), **kw})


@pytest.mark.parametrize("cfg,page", [(TINY_A, 8), (TINY_C, 16), (TINY_D, 16), (TINY_E, 5)])
def test_a_text_with_a_bounded_cache(tmp_path, cfg, page):
    cfg = all_keys(cfg)
    d = helpers.make_model(tmp_path, cfg, 3)
    raw, w = plain_impl.load_folder(d)
    v = cfg["vocab_size"]
    eng = engine(d, page_size=page)
    # many steps of single tokens of all requests: recorded, and replayed across evictions
    cuts = cases.bounded_run(eng, lambda name: cases.PlainBounded(raw, w), text(330, v), [40, 133, 1, 1, 1, 100] + [1] * 20, 60, 12, 4, 20,
                             others=[("short", text(40, v, 1), [5, 1, 1, 1, 1] + [1] * 20), ("long", text(300, v, 2), [160, 1, 1, 1, 1, 66] + [1] * 20)])
    assert cuts >= 5 and eng.graph_replays > 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_recorded_steps_of_many_requests_count_every_query_once(tmp_path, dtype):
    """Batches that a recorded step would fill up with copies of their last entry are not filled here."""
    cfg = all_keys(TINY_E)
    d = helpers.make_model(tmp_path, cfg, 3, torch.bfloat16)
    eng, v = engine(d, dtype), cfg["vocab_size"]
    n = 7
    eng.step([StepEntry(i, text(20 + i, v, i), []) for i in range(n)])
    for k in range(6):
        eng.step([StepEntry(i, text(1, v, 100 + k), [0]) for i in range(n)])
    assert eng.graph_replays > 0
    group = eng.cache.groups[0]
    for i in range(n):
        c = eng.cache.cached_len(i)
        for layer in range(2):
            rows = group.data["mass"][layer][eng.cache.block_table(i, 0)][:, :, :, 0].transpose(0, 1).reshape(1, -1)[:, :c]
            assert abs(float(rows.double().sum()) - c * 7) < c * 7 * 1e-4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_evictions_do_not_depend_on_the_pages(tmp_path, dtype):
    cfg = all_keys(TINY_D)
    d = helpers.make_model(tmp_path, cfg, 5, torch.bfloat16)
    v = cfg["vocab_size"]

    def run(**kw):
        eng, out = engine(d, dtype, **kw), []
        eng.step([StepEntry("other", text(30, v, 9), [])])
        for n, seed in ((200, 0), (1, 1), (1, 2), (1, 3), (90, 4), (1, 5), (1, 6)):
            out.append(eng.step([StepEntry("r", text(n, v, seed), [n - 1])]).clone())
            eng.evict(["r"], 64, first=2, recent=16)
            assert eng.cache.cached_len("r") <= 64
        eng.cache.check_invariants()
        return torch.cat(out)
    a = run()
    for kw in (dict(page_order_seed=7), dict(page_order_seed=None, num_pages=700, max_tokens=None)):
        assert torch.equal(a, run(**kw))
    # tables of another width: the attention cuts a token's keys at other places, so its sums run in another order (in float32 some
    # hundred roundings of 2^-24 a layer; in bfloat16 a rounding of 2^-8 that falls the other way, a few of them on the way through two layers)
    for kw in (dict(use_graphs=False), dict(page_size=32)):
        assert float((a - run(**kw)).abs().max()) <= (1e-4 if dtype == "float32" else 0.05) * float(a.abs().max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_without_an_eviction_the_sums_change_nothing(tmp_path, dtype):
    cfg = all_keys(TINY_E)
    d = helpers.make_model(tmp_path, cfg, 4, torch.bfloat16)
    v = cfg["vocab_size"]
    a, b = engine(d, dtype), engine(d, dtype, attention_mass=False)
    for n in (70, 1, 1, 1, 40):
        part = text(n, v, n)
        assert torch.equal(a.step([StepEntry("r", part, [n - 1])]), b.step([StepEntry("r", part, [n - 1])]))


@pytest.mark.parametrize("lookahead", [False, True])
def test_a_scheduler_with_a_budget(tmp_path, lookahead):
    cfg = all_keys(TINY_D)
    d = helpers.make_model(tmp_path, cfg, 5, torch.bfloat16)
    v = cfg["vocab_size"]
    eng = engine(d, "bfloat16", max_tokens=700, max_seqs=8)
    sched = Scheduler(eng, chunk_size=96, max_batch_tokens=256, cache_budget=64, cache_slack=16, lookahead=lookahead)
    prompts = {i: text(n, v, i) for i, n in enumerate((500, 20, 333, 61, 90, 400))}
    for rid, p in prompts.items():
        sched.add_request(p, 40, rid=rid, logprobs=4 if rid % 2 else None)
    while sched.has_unfinished():
        sched.step()
        assert all(eng.cache.cached_len(r) <= 80 for r in eng.cache.live())
    eng.cache.check_invariants()
    for rid in prompts:
        rows = sched.requests[rid].logprobs
        assert len(sched.output(rid)) == 40 and len(rows) == (40 if rid % 2 else 0)
        for r, tok in zip(rows, sched.output(rid)):
            assert r.token == tok == r.top[0][0] and r.logprob == r.top[0][1] and len(r.top) == 4          # (greedy)


def test_score(tmp_path):
    cfg = all_keys(TINY_A)
    d = helpers.make_model(tmp_path, cfg, 3)
    raw, w = plain_impl.load_folder(d)
    m = Qwen2(d, dtype="float32", page_size=8, max_tokens=1024, max_seqs=2, chunk_size=64)
    toks = text(300, cfg["vocab_size"])
    y = torch.log_softmax(torch.from_numpy(plain_impl.forward(raw, w, toks)), 1)[:-1]
    rows = m.score(toks, top=5)
    assert [r.token for r in rows] == toks[1:]
    want, entropy = y.gather(1, torch.tensor(toks[1:])[:, None])[:, 0].tolist(), (-(y.exp() * y).sum(1)).tolist()
    assert max(abs(r.logprob - a) for r, a in zip(rows, want)) < 1e-4 and max(abs(r.entropy - a) for r, a in zip(rows, entropy)) < 1e-4
    top = torch.sort(y, dim=1, descending=True).values[:, :5].tolist()
    assert max(abs(v - e) for r, t in zip(rows, top) for (_, v), e in zip(r.top, t)) < 1e-4


@pytest.mark.parametrize("chunk", [64, 7])
def test_score_with_windowed_layers(tmp_path, chunk):
    d = helpers.make_model(tmp_path, TINY_B, 3)
    raw, w = plain_impl.load_folder(d)
    m = Qwen2(d, dtype="float32", page_size=8, max_tokens=1024, max_seqs=2, chunk_size=chunk)
    toks = text(120, raw["vocab_size"])
    y = torch.log_softmax(torch.from_numpy(plain_impl.forward(raw, w, toks)), 1)[:-1]
    rows = m.score(toks)
    want = y.gather(1, torch.tensor(toks[1:])[:, None])[:, 0].tolist()
    assert len(rows) == 119 and max(abs(r.logprob - a) for r, a in zip(rows, want)) < 1e-4


def test_two_engines_take_turns(tmp_path):
    """Two models in one process, steps and evictions in turn on one stream."""
    ds = [helpers.make_model(tmp_path, all_keys(c), 3, name=n) for c, n in ((TINY_A, "a"), (TINY_D, "d"))]
    loaded = [plain_impl.load_folder(d) for d in ds]
    engines = [engine(d) for d in ds]
    refs = [cases.PlainBounded(*l) for l in loaded]
    for n in (90, 1, 1, 1, 60, 1, 1):
        for e, r, (raw, _) in zip(engines, refs, loaded):
            part = text(n, raw["vocab_size"], n)
            got, want = e.step([StepEntry("x", part, list(range(n)))]).cpu().double().numpy(), r.step(part)
            assert np.abs(got - want).max() <= 2e-5 * np.abs(want).max()
            e.evict(["x"], 40)
            r.evict(40)
