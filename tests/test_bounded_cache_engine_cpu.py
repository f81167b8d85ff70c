"""The engine, the scheduler and the entry point around a cache of bounded length and around log probabilities, with stand-ins for
the kernels: bookkeeping, positions, what is refused.  The GPU twin is tests/test_bounded_cache_engine_gpu.py."""
import math

import numpy as np
import pytest
import torch

import bounded_cache_cases as cases
import helpers
import plain_impl
from litinfer_amd.cache import CacheManager
from litinfer_amd.engine import Engine, Scheduler, StepEntry
from litinfer_amd.kernels import ops
from litinfer_amd.models import Qwen2
from litinfer_amd.parts import PagedKVNeed, PagedNeed, PagedTensor
from litinfer_amd.sampling import SamplingParams
from tiny_configs import TINY_A, TINY_B

CFG = {**TINY_A, "max_position_embeddings": 512}


@pytest.fixture
def bounded_ops(cpu_ops, monkeypatch):
    for f in cases.STAND_INS:
        monkeypatch.setattr(ops, f.__name__, f)


@pytest.fixture
def model(tmp_path):
    return helpers.make_model(tmp_path, CFG, 3)


def engine(d, **kw):
    return Engine.from_dir(d, **{**dict(dtype="float32", device="cpu", page_size=8, max_seqs=4, max_tokens=600, attention_mass=True, page_order_seed=1), **kw})


def text(n, seed=0, vocab=CFG["vocab_size"]):
    return np.random.default_rng(seed).integers(0, vocab, n).tolist()


# ------------------------------------------------------------------------------------------------- the book
def manager(**kw):
    need = PagedNeed(PagedKVNeed(2, 4).tensors + (PagedTensor("mass", (2, 1), torch.float32, accumulates=True),))
    return CacheManager([need], [None], **{**dict(page_size=4, num_pages=10, max_seqs=3, dtype=torch.float32, device="cpu"), **kw})


def test_the_book_after_an_eviction():
    c = manager()
    c.admit("a"), c.admit("b")
    for rid, n in (("a", 19), ("b", 6)):
        c.reserve(rid, n)
        c.commit(rid, n)
    table = c.block_table("a", 0)
    c.reserve("a", 3)                                             # (a page for tokens that never came goes back too)
    c.evict_many(c.handles_of(["a"]), 9)
    assert c.cached_len("a") == 9 and c.block_table("a", 0) == table[:3] and c.free_pages() == [10 - 3 - 2]
    assert c.positions_many(c.handles_of(["a", "b"])).tolist() == [19, 6]
    c.check_invariants()
    c.reserve("a", 4)
    c.commit("a", 4)
    assert c.cached_len("a") == 13 and c.positions_many(c.handles_of(["a"])).tolist() == [23] and c.table_len("a", 0) == 4
    c.evict_many(c.handles_of(["a", "b"]), 6)
    assert c.positions_many(c.handles_of(["a", "b"])).tolist() == [23, 6] and [c.cached_len(r) for r in "ab"] == [6, 6]
    c.check_invariants()
    c.release("a")
    c.admit("a")
    assert c.positions_many(c.handles_of(["a"])).tolist() == [0]


def test_the_book_refuses_evictions_that_make_no_sense():
    c = manager()
    c.admit("a")
    c.reserve("a", 5)
    c.commit("a", 5)
    for keep in (0, -1, 6):
        with pytest.raises(ValueError, match="cache:"):
            c.evict_many(c.handles_of(["a"]), keep)
    with pytest.raises(ValueError, match="unknown"):
        c.evict_many(np.array([99], dtype=np.int64), 2)
    assert c.cached_len("a") == 5
    with pytest.raises(ValueError, match="add to"):
        c.rewind("a", 1)
    c.rewind("a", 0)
    windowed = CacheManager([PagedKVNeed(2, 4, 16)], [None], page_size=4, num_pages=10, max_seqs=2, dtype=torch.float32, device="cpu")
    windowed.admit("a")
    windowed.reserve("a", 5)
    windowed.commit("a", 5)
    with pytest.raises(ValueError, match="windowed"):
        windowed.evict_many(windowed.handles_of(["a"]), 3)


# ------------------------------------------------------------------------------------------------- the engine
def test_a_text_with_a_bounded_cache(bounded_ops, model):
    cfg, w = plain_impl.load_folder(model)
    eng = engine(model)
    cuts = cases.bounded_run(eng, lambda name: cases.PlainBounded(cfg, w), text(150), [40, 33, 1, 1, 1, 40, 1, 1, 20, 1, 1, 10], 24, 8, 4, 10,
                             others=[("short", text(20, 1), [5, 1, 1, 1, 12]), ("long", text(90, 2), [60, 1, 1, 1, 1, 26])])
    assert cuts >= 6


def test_more_tokens_than_the_cache_could_hold(bounded_ops, model):
    eng = engine(model, max_tokens=64)
    toks = text(400)
    for at in range(0, 400, 16):
        eng.step([StepEntry("r", toks[at:at + 16], [15])])
        eng.evict(["r"], 20)
    assert eng.cache.cached_len("r") == 20
    eng.step([StepEntry("r", text(20, 5), [0])])
    eng.evict(["r"], 20)
    with pytest.raises(ValueError, match="max sequence length is 512"):       # (positions go on where they were)
        eng.step([StepEntry("r", text(93, 6), [0])])
    eng.step([StepEntry("r", text(30, 6), [0])])


def test_without_an_eviction_the_sums_change_nothing(bounded_ops, model):
    toks = text(60)
    a, b = engine(model), engine(model, attention_mass=False)
    for part in (toks[:40], toks[40:41], toks[41:]):
        want = list(range(len(part)))
        assert torch.equal(a.step([StepEntry("r", part, want)]), b.step([StepEntry("r", part, want)]))
    assert a.evict(["r"], 60) == [60] and a.evict(["r"], 1000) == [60]
    # every query has given one unit a head
    mass = a.cache.groups[0].data["mass"]
    table = a.cache.block_table("r", 0)
    for layer in range(mass.shape[0]):
        rows = mass[layer][table].transpose(1, 2).reshape(-1, 2)[:60]
        assert abs(float(rows.sum()) - 60 * 4) < 60 * 4 * 1e-5


def test_the_engine_refuses(bounded_ops, model, tmp_path):
    eng = engine(model)
    eng.step([StepEntry("r", text(30), [])])
    for bad in (dict(keep=0), dict(keep=-3), dict(keep=5, first=-1), dict(keep=5, recent=-1)):
        with pytest.raises(ValueError, match="evict"):
            eng.evict(["r"], **bad)
    with pytest.raises(ValueError, match="twice"):
        eng.evict(["r", "r"], 5)
    with pytest.raises(KeyError):
        eng.evict(["r", "nobody"], 5)
    assert eng.cache.cached_len("r") == 30
    plain = engine(model, attention_mass=False)
    plain.step([StepEntry("r", text(30), [])])
    with pytest.raises(ValueError, match="attention_mass"):
        plain.evict(["r"], 5)
    windowed = helpers.make_model(tmp_path, TINY_B, 1, name="windowed")
    with pytest.raises(ValueError, match="attend over all"):
        Engine.from_dir(windowed, dtype="float32", device="cpu", max_tokens=64, attention_mass=True)


@pytest.mark.parametrize("design", ["sogenex", "besorax", "dimelix", "nusuvik", "tovasun", "kufolorn"])
def test_models_with_other_caches_are_refused(bounded_ops, design):
    from litinfer_amd import benchmark
    from litinfer_amd.config import architecture_name, lookup
    cfg = getattr(benchmark, design + "_config")("1.5b", 4)
    arch = lookup(architecture_name(cfg))
    with pytest.raises(ValueError, match="attend over all"):
        from litinfer_amd.engine.engine import Engine as E
        E(arch.model_spec(arch.config_from_dict(cfg)), device="cpu", dtype="float32", attention_mass=True)


# --------------------------------------------------------------------------------------- scheduler and entry point
@pytest.mark.parametrize("lookahead", [False, True])
def test_requests_with_a_budget_run_in_a_pool_that_could_not_hold_them(bounded_ops, model, lookahead):
    eng = engine(model, max_tokens=160, max_seqs=3)
    sched = Scheduler(eng, chunk_size=32, max_batch_tokens=64, cache_budget=24, cache_slack=8, lookahead=lookahead)
    prompts = {f"r{i}": text(n, i) for i, n in enumerate((100, 7, 150, 60))}
    for rid, p in prompts.items():
        sched.add_request(p, 30, rid=rid)
    worst = 0
    while sched.has_unfinished():
        sched.step()
        worst = max([worst] + [eng.cache.cached_len(r) for r in eng.cache.live()])
        eng.cache.check_invariants()
    assert worst <= 24 + 8 and all(len(sched.output(r)) == 30 for r in prompts)
    # each alone, through the engine: the same cuts and the same tokens
    for rid, p in prompts.items():
        alone = Scheduler(engine(model), chunk_size=32, max_batch_tokens=64, cache_budget=24, cache_slack=8)
        one = alone.add_request(p, 30)
        alone.run_to_completion()
        if len(p) <= 32:                                          # (longer prompts are cut into portions by what else is in a step)
            assert alone.output(one) == sched.output(rid)


def test_a_scheduler_without_a_budget_refuses_what_one_with_a_budget_takes(bounded_ops, model):
    eng = engine(model, max_tokens=64)
    with pytest.raises(ValueError, match="never run"):
        Scheduler(eng, chunk_size=16).add_request(text(100), 10)
    sched = Scheduler(eng, chunk_size=16, cache_budget=24, cache_slack=8)
    rid = sched.add_request(text(100), 10)
    sched.run_to_completion()
    assert len(sched.output(rid)) == 10 and sched.requests[rid].finish_reason == "length"
    for bad in (dict(cache_budget=0), dict(cache_budget=-1), dict(cache_budget=5, cache_slack=-1)):
        with pytest.raises(ValueError, match="cache_budget"):
            Scheduler(eng, **bad)
    with pytest.raises(ValueError, match="cache_budget"):
        Scheduler(engine(model, attention_mass=False), cache_budget=24)


def expected_rows(cfg, w, tokens, start):
    """(log probability, entropy) of tokens[i] for i >= start, and all log probabilities there."""
    y = torch.log_softmax(torch.from_numpy(plain_impl.forward(cfg, w, tokens)[start - 1:-1]), 1)
    return y.gather(1, torch.tensor(tokens[start:])[:, None])[:, 0], -(y.exp() * y).sum(1), y


@pytest.mark.parametrize("lookahead", [False, True])
def test_log_probabilities_of_generated_tokens(bounded_ops, model, lookahead):
    cfg, w = plain_impl.load_folder(model)
    sched = Scheduler(engine(model), chunk_size=16, lookahead=lookahead)
    asked = {"a": (None, None), "b": (0, None), "c": (3, SamplingParams(temperature=0.8, top_k=20, seed=5)), "d": (7, None)}
    prompts = {rid: text(10 + 9 * i, i) for i, rid in enumerate(asked)}
    for rid, (n, params) in asked.items():
        sched.add_request(prompts[rid], 6, params, rid=rid, logprobs=n)
    sched.run_to_completion()
    for rid, (n, _) in asked.items():
        rows, out = sched.requests[rid].logprobs, sched.output(rid)
        if n is None:
            assert rows == []
            continue
        assert [r.token for r in rows] == out and len(out) == 6
        lp, ent, y = expected_rows(cfg, w, prompts[rid] + out, len(prompts[rid]))
        for r, a, b, row in zip(rows, lp.tolist(), ent.tolist(), y):
            assert abs(r.logprob - a) < 1e-4 and abs(r.entropy - b) < 1e-4 and len(r.top) == n
            order = torch.sort(row, descending=True, stable=True)
            assert [i for i, _ in r.top] == order.indices[:n].tolist()
            assert all(abs(v - e) < 1e-4 for (_, v), e in zip(r.top, order.values.tolist()))
    for bad in (-1, 33, 2.5, True, "3"):
        with pytest.raises(ValueError, match="alternatives"):
            sched.add_request([1, 2], 2, logprobs=bad)


def test_a_sampler_without_log_probabilities_is_refused_when_they_are_asked_for(bounded_ops, model):
    class Own:
        def sample(self, logits, params, counters):
            return [0] * logits.shape[0]
    sched = Scheduler(engine(model), sampler=Own())
    with pytest.raises(ValueError, match="no log probabilities"):
        sched.add_request([1, 2], 2, logprobs=0)
    rid = sched.add_request([1, 2], 2)
    sched.run_to_completion()
    assert sched.output(rid) == [0, 0]


def test_log_probabilities_of_a_preempted_request(bounded_ops, model):
    def run(**kw):
        sched = Scheduler(engine(model, **kw), chunk_size=16)
        for i in range(3):
            sched.add_request(text(20, i), 30, rid=i, logprobs=2)
        sched.run_to_completion()
        return sched
    a, b = run(max_tokens=96), run(max_tokens=600)
    assert a.preemptions > 0 and b.preemptions == 0
    for i in range(3):
        assert a.output(i) == b.output(i) and len(a.requests[i].logprobs) == 30
        assert all(x.token == y.token and abs(x.logprob - y.logprob) < 1e-4 for x, y in zip(a.requests[i].logprobs, b.requests[i].logprobs))


def test_an_end_token_leaves_no_log_probability(bounded_ops, model):
    sched = Scheduler(engine(model), chunk_size=16, lookahead=True)
    rid = sched.add_request(text(12), 8, logprobs=1)
    sched.run_to_completion()
    out = sched.output(rid)
    ending = Scheduler(engine(model), chunk_size=16, eos_token_ids=[out[3]], lookahead=True)
    rid = ending.add_request(text(12), 8, logprobs=1)
    ending.run_to_completion()
    want = out[:out.index(out[3])]
    assert ending.output(rid) == want and [r.token for r in ending.requests[rid].logprobs] == want


def test_score(bounded_ops, model, capsys):
    cfg, w = plain_impl.load_folder(model)
    m = Qwen2(model, device="cpu", dtype="float32", page_size=8, max_tokens=256, max_seqs=2, chunk_size=16)
    toks = text(70)
    rows = m.score(toks, top=2)
    lp, ent, y = expected_rows(cfg, w, toks, 1)
    assert [r.token for r in rows] == toks[1:]
    assert max(abs(r.logprob - a) for r, a in zip(rows, lp.tolist())) < 1e-4 and max(abs(r.entropy - a) for r, a in zip(rows, ent.tolist())) < 1e-4
    assert [r.top[0][0] for r in rows] == y.argmax(1).tolist()
    assert m.engine.cache.live() == [] and m.score([5]) == []
    for bad in ([], [1, 256], [-1, 4], [1] * 600):
        with pytest.raises(ValueError, match="score"):
            m.score(bad)
    with pytest.raises(ValueError, match="score"):
        m.score([1, 2], top=99)
    # the same text with a cache that is cut between the portions
    ref, want = cases.PlainBounded(cfg, w), []
    short = Qwen2(model, device="cpu", dtype="float32", page_size=8, max_tokens=256, max_seqs=2, chunk_size=100, cache_budget=40)
    long = text(500, 9)
    for at in range(0, 499, 100):
        part = long[at:min(at + 100, 499)]
        y = torch.log_softmax(torch.from_numpy(ref.step(part)), 1)
        want += y.gather(1, torch.tensor(long[at + 1:at + 1 + len(part)])[:, None])[:, 0].tolist()
        if ref.cached > 40 + 128:
            ref.evict(40)
    got = short.score(long)
    assert max(abs(r.logprob - a) for r, a in zip(got, want)) < 1e-4
    short.engine_start()
    rid = short.engine_add_request(long[:300], 5, logprobs=1)
    while short.engine_has_unfinished():
        short.engine_step()
    assert [r.token for r in short.engine_get_logprobs(rid)] == short.engine_get_output(rid)


def test_score_on_the_command_line(bounded_ops, model, capsys):
    import json
    from litinfer_amd.__main__ import main
    toks = text(30)
    assert main(["score", "--model", str(model), "--device", "cpu", "--dtype", "float32", "--num-pages", "20", "--prompt-ids", ",".join(map(str, toks)), "--top", "2"]) == 0
    out = json.loads(capsys.readouterr().out.splitlines()[-1])
    cfg, w = plain_impl.load_folder(model)
    lp, _, _ = expected_rows(cfg, w, toks, 1)
    assert out["tokens"] == 29 and abs(out["logprob"] - float(lp.sum())) < 1e-3 and abs(out["perplexity"] - math.exp(-float(lp.mean()))) < 0.5
    assert [r["token"] for r in out["rows"]] == toks[1:] and all(len(r["top"]) == 2 for r in out["rows"])
    assert main(["generate", "--model", str(model), "--device", "cpu", "--dtype", "float32", "--num-pages", "40", "--prompt-ids", ",".join(map(str, text(200))), "--max_steps", "3",
                 "--test", "--cache-budget", "50"]) == 0
    assert len(json.loads(capsys.readouterr().out.splitlines()[-1])["tokens"]) == 3


def test_a_perplexity_beyond_all_numbers():
    from litinfer_amd.__main__ import _perplexity
    assert _perplexity(-math.log(8.0) * 5, 5) == pytest.approx(8.0, rel=1e-12)
    assert _perplexity(-1e5, 3) == math.inf and _perplexity(-math.inf, 3) == math.inf and _perplexity(0.0, 0) is None
    assert math.isnan(_perplexity(math.nan, 2))


def test_score_goes_by_the_largest_step(bounded_ops, model):
    m = Qwen2(model, device="cpu", dtype="float32", page_size=8, max_tokens=256, max_seqs=2, chunk_size=64, max_batch_tokens=24)
    sizes, step = [], m.engine.step
    m.engine.step = lambda entries: sizes.append(sum(len(e.tokens) for e in entries)) or step(entries)
    rows = m.score(text(71))
    assert len(rows) == 70 and sizes == [24, 24, 22]


@pytest.mark.parametrize("bad", [dict(cache_budget=0), dict(cache_slack=-1), dict(cache_first=-1), dict(cache_recent=-2)])
def test_a_scheduler_refuses_budgets_that_make_no_sense(bounded_ops, model, bad):
    with pytest.raises(ValueError, match="cache_budget"):
        Scheduler(engine(model), **{"cache_budget": 16, **bad})
