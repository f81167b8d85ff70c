"""Requests with a bounded cache, and texts that are scored, in pools that hold little more than they need (stand-ins for the kernels)."""
import json
import math

import numpy as np
import pytest
import torch

import bounded_cache_cases as cases
import helpers
import plain_impl
from litinfer_amd.cache import CacheFull
from litinfer_amd.engine import Engine, Scheduler, StepEntry
from litinfer_amd.engine.workspace import Workspace
from litinfer_amd.kernels import ops
from litinfer_amd.models import Qwen2
from litinfer_amd.sampling import Sampler, TokenLogprob
from tiny_configs import TINY_A, TINY_B

CFG = {**TINY_A, "max_position_embeddings": 512}


@pytest.fixture
def bounded_ops(cpu_ops, monkeypatch):
    for f in cases.STAND_INS:
        monkeypatch.setattr(ops, f.__name__, f)


@pytest.fixture
def model(tmp_path):
    return helpers.make_model(tmp_path, CFG, 3)


def text(n, seed=0, vocab=CFG["vocab_size"]):
    return np.random.default_rng(seed).integers(0, vocab, n).tolist()


def steps_of(eng):
    """The numbers of tokens of the steps that the engine takes from now on."""
    sizes, step = [], eng.step
    eng.step = lambda entries: sizes.append(sum(len(e.tokens) for e in entries)) or step(entries)
    return sizes


# -------------------------------------------------------------------------------------------------- score
def check_scored_in(model, toks, rows, sizes, budget, slack):
    """The rows are those of the text in portions of `sizes`, its cache cut to `budget` where it has outgrown the slack."""
    cfg, w = plain_impl.load_folder(model)
    ref, at, want = cases.PlainBounded(cfg, w), 0, []
    for n in sizes:
        y = torch.log_softmax(torch.from_numpy(ref.step(toks[at:at + n])), 1)
        want += y.gather(1, torch.tensor(toks[at + 1:at + 1 + n])[:, None])[:, 0].tolist()
        at += n
        if ref.cached > budget + slack:
            ref.evict(budget)
    assert at == len(toks) - 1 and [r.token for r in rows] == toks[1:]
    assert max(abs(r.logprob - a) for r, a in zip(rows, want)) < 1e-4


@pytest.mark.parametrize("pages", [22, 24, 28, 40])
def test_score_takes_portions_that_fit_the_pool(bounded_ops, model, pages):
    """budget 40, slack 128, portions of 64: 22 pages of 8 hold budget and slack and a token, 29 a whole portion too."""
    m = Qwen2(model, device="cpu", dtype="float32", page_size=8, num_pages=pages, max_seqs=2, chunk_size=64, cache_budget=40)
    toks = text(400)
    assert len(m.generate(toks, max_new_tokens=3)) == 3
    sizes = steps_of(m.engine)
    rows = m.score(toks)
    check_scored_in(model, toks, rows, sizes, 40, 128)
    assert max(sizes) == 64 and (min(sizes[:-1]) < 64) == (pages < 29)
    assert m.engine.cache.live() == [] and m.engine.cache.free_pages() == [pages]


def test_score_beside_requests_that_hold_pages(bounded_ops, model):
    m = Qwen2(model, device="cpu", dtype="float32", page_size=8, num_pages=30, max_seqs=3, chunk_size=64, cache_budget=40)
    m.engine_start()
    rid = m.engine_add_request(text(60, 5), 6)
    m.engine_step()
    held = len(m.engine.cache.block_table(rid, 0))
    sizes = steps_of(m.engine)
    toks = text(300, 1)
    check_scored_in(model, toks, m.score(toks), sizes, 40, 128)
    assert held == 8 and min(sizes[:-1]) < 64
    while m.engine_has_unfinished():
        m.engine_step()
    assert len(m.engine_get_output(rid)) == 6


def test_score_of_a_text_that_does_not_fit_at_all(bounded_ops, model):
    m = Qwen2(model, device="cpu", dtype="float32", page_size=8, num_pages=10, max_seqs=2, chunk_size=64)
    with pytest.raises(CacheFull):
        m.score(text(100))
    assert m.engine.cache.live() == [] and m.engine.cache.free_pages() == [10]
    assert len(m.score(text(81))) == 80


def test_score_with_windowed_layers_in_a_pool_of_little_more_than_the_window(bounded_ops, tmp_path):
    d = helpers.make_model(tmp_path, TINY_B, 3, name="windowed")
    raw, w = plain_impl.load_folder(d)
    toks = text(100, 2, raw["vocab_size"])
    y = torch.log_softmax(torch.from_numpy(plain_impl.forward(raw, w, toks)), 1)[:-1]
    want = y.gather(1, torch.tensor(toks[1:])[:, None])[:, 0].tolist()
    whole = Qwen2(d, device="cpu", dtype="float32", page_size=8, max_tokens=256, max_seqs=2, chunk_size=64)
    window = max(g.need.reach for g in whole.engine.cache.groups)
    assert window > 0
    pages = [13 if g.need.reach <= 0 else -(-window // 8) + 2 for g in whole.engine.cache.groups]
    m = Qwen2(d, device="cpu", dtype="float32", page_size=8, num_pages=pages, max_seqs=2, chunk_size=64)
    sizes = steps_of(m.engine)
    rows = m.score(toks)
    assert max(abs(r.logprob - a) for r, a in zip(rows, want)) < 1e-4 and max(sizes) < 64


@pytest.mark.parametrize("top", [None, -1, 33, True, 1.5])
def test_score_refuses_numbers_of_alternatives(bounded_ops, model, top):
    m = Qwen2(model, device="cpu", dtype="float32", page_size=8, num_pages=30, max_seqs=2)
    with pytest.raises(ValueError, match="score: the number of alternatives"):
        m.score(text(9), top=top)
    with pytest.raises(ValueError, match="logprobs: the number of alternatives"):
        Sampler("cpu").logprobs_async(torch.zeros(2, 99), torch.zeros(2, dtype=torch.int32), top)


def test_what_score_prints_is_json_whatever_the_numbers_are(bounded_ops, model, monkeypatch, capsys):
    def score(self, ids, top=0):
        return [TokenLogprob(7, -math.inf, 0.5, ((3, -0.25), (4, -math.inf))), TokenLogprob(8, math.nan, math.nan, ((3, math.nan), (4, math.nan))), TokenLogprob(9, -1e5, 1.0, ())]
    monkeypatch.setattr(Qwen2, "score", score)
    from litinfer_amd.__main__ import main
    assert main(["score", "--model", str(model), "--device", "cpu", "--dtype", "float32", "--num-pages", "20", "--prompt-ids", "1,2,3,4"]) == 0

    def refuse(name):
        raise AssertionError(name)
    out = json.loads(capsys.readouterr().out.splitlines()[-1], parse_constant=refuse)
    assert out["logprob"] is None and out["perplexity"] is None
    assert [r["logprob"] for r in out["rows"]] == [None, None, -1e5] and [r["entropy"] for r in out["rows"]] == [0.5, None, 1.0]
    assert [r["top"] for r in out["rows"]] == [[[3, -0.25], [4, None]], [[3, None], [4, None]], []]


# ---------------------------------------------------------------------------------------------- scheduler
def engine(d, **kw):
    return Engine.from_dir(d, **{**dict(dtype="float32", device="cpu", page_size=8, max_seqs=4, attention_mass=True, page_order_seed=1), **kw})


def run_two(model, pages, steps_before):
    """Two prompts of 200, the second some steps after the first: how many steps both were running, the most pages that were held."""
    eng = engine(model, num_pages=pages)
    sched = Scheduler(eng, chunk_size=16, max_batch_tokens=64, cache_budget=24, cache_slack=8)
    sched.add_request(text(200), 4, rid="a")
    for _ in range(steps_before):
        sched.step()
    sched.add_request(text(200, 1), 4, rid="b")
    both = 0
    while sched.has_unfinished():
        sched.step()
        eng.cache.check_invariants()
        both += len(sched.running) == 2
    assert sched.preemptions == 0 and [len(sched.output(r)) for r in "ab"] == [4, 4]
    return both


@pytest.mark.parametrize("steps_before", [1, 2, 3, 5])
def test_a_second_long_prompt_runs_beside_the_first_in_a_pool_of_two_peaks(bounded_ops, model, steps_before):
    """A request holds at most ceil((24 + 8 + 16) / 8) = 6 pages at a time: what the first holds already is part of its six."""
    assert run_two(model, 12, steps_before) >= 13 - steps_before - 1
    assert run_two(model, 11, steps_before) <= 5                  # one page less: the second waits for the end of the first prompt (its last portion, four tokens)


def test_what_a_windowed_request_holds_does_not_count_against_what_it_takes(bounded_ops, tmp_path):
    """Without a budget nothing has changed: the windowed group's cap is what has to be free."""
    d = helpers.make_model(tmp_path, TINY_B, 3, name="windowed")
    sched = Scheduler(Engine.from_dir(d, dtype="float32", device="cpu", page_size=8, max_seqs=2, max_tokens=256))
    need = np.full((2, len(sched.cache.groups)), 1000, dtype=np.int32)
    held = np.full_like(need, 3)
    assert (sched._at_a_time(need) == sched._at_a_time(need, held=held)).all()


@pytest.mark.parametrize("bad", [dict(cache_budget=0.5), dict(cache_budget=24.0), dict(cache_budget=True), dict(cache_budget="24"), dict(cache_slack=1.5), dict(cache_first=2.0),
                                 dict(cache_recent=0.5), dict(cache_recent=math.nan), dict(cache_budget=math.inf)])
def test_budgets_that_are_no_whole_numbers_are_refused_before_anything_runs(bounded_ops, model, bad):
    with pytest.raises(ValueError, match="cache_budget"):
        Scheduler(engine(model, num_pages=20), **{"cache_budget": 16, **bad})


@pytest.mark.parametrize("bad", [0, -3, 0.5, 24.0, True, "24"])
def test_the_entry_point_refuses_such_a_budget_before_it_loads_anything(bounded_ops, tmp_path, bad):
    with pytest.raises(ValueError, match="cache_budget"):
        Qwen2(tmp_path / "nothing is here", device="cpu", cache_budget=bad)


def test_budgets_of_numpy_are_whole_numbers_too(bounded_ops, model):
    sched = Scheduler(engine(model, num_pages=20), chunk_size=16, cache_budget=np.int64(24), cache_slack=np.int32(8), cache_recent=np.int16(4))
    rid = sched.add_request(text(100), 2)
    sched.run_to_completion()
    assert len(sched.output(rid)) == 2


# ---------------------------------------------------------------------------------------------- workspace
def work_floats(q_len, ctx_len, nh, nkv, dh=64, padded=0):
    q, c = np.asarray(q_len, dtype=np.int32), np.asarray(ctx_len, dtype=np.int32)
    return ops._mass_work_floats()(q.ctypes.data, c.ctypes.data, len(q), int(q.sum()), padded, nh, nkv, dh, ops._DT[torch.bfloat16], (nh + 2 * nkv) * dh, 1 << 20, 1 << 20,
                                   0.125, 1 << 20)


ROOM = 1 << 26                                                    # floats that requests take together


def scores(nh, ctx):
    """What a request's scores take in runs of 64 keys, and a run's statistics, 16 of them in a line."""
    runs = -(-ctx // 64)
    return nh * (64 * runs + 2 * 16 * -(-runs // 16))


def test_the_workspace_of_single_tokens_goes_by_what_each_has_cached():
    ctx = [100] * 63 + [32000]
    assert work_floats([1] * 64, ctx, 28, 4) == sum(scores(28, c) for c in ctx) < 1.1 * 28 * sum(ctx) * 66 / 64
    assert work_floats([1, 40, 1], [500, 90, 70000], 28, 4) - work_floats([40], [90], 28, 4) <= scores(28, 500) + scores(28, 70000) + 4096


@pytest.mark.parametrize("n,nh,nkv,longest", [(64, 40, 8, 32768), (256, 40, 8, 131072), (1000, 28, 4, 4096), (3, 64, 8, 1 << 20)])
def test_the_workspace_of_single_tokens_has_a_bound(n, nh, nkv, longest):
    most = max(ROOM, scores(nh, longest))
    assert work_floats([1] * n, [9] * n, nh, nkv, padded=longest) <= most               # a recorded step: any length up to the tables'
    assert work_floats([1] * n, [longest] * n, nh, nkv) <= most


def test_the_workspace_of_a_request_that_takes_more_than_the_room_by_itself():
    assert work_floats([1] * 3, [5000, 4 << 20, 5000], 64, 8) == scores(64, 4 << 20) > ROOM
    assert work_floats([1] * 3, [9] * 3, 64, 8, padded=4 << 20) == scores(64, 4 << 20)


def test_batches_of_many_sizes_ask_the_workspace_for_few(monkeypatch):
    monkeypatch.setattr(ops, "_here", lambda what, *ts: None)
    asked = []
    monkeypatch.setattr(ops, "_run", lambda module, name, *args: asked.append(args))
    ws, rng = Workspace("cpu"), np.random.default_rng(3)
    for _ in range(400):
        segs = [(int(q), int(q + c)) for q, c in zip(rng.choice([1, 1, 1, 7, 40], 5), rng.integers(0, 3000, 5))]
        meta, pages = cases.batch(segs, 16, "cpu")
        ops.attention_mass(torch.zeros(meta.num_tokens, 12 * 64), torch.zeros(pages, 2, 16, 1), torch.zeros(pages, 2, 16, 64), meta, 8, 2, 64, 16, 0.125, ws=ws)
    sizes = [args[-1] for args in asked]
    assert len(sizes) == 400
    # eight sizes between two powers of two, and an eighth more at most
    octaves = math.log2(max(sizes) / min(sizes)) + 1
    assert len(ws._views) <= len(set(sizes)) <= 8 * octaves + 1 and ws.generation <= 2 * octaves


def test_what_the_sums_take_is_set_aside_before_the_pages_are_counted(bounded_ops, model):
    a, b = engine(model, num_pages=10), engine(model, num_pages=10, attention_mass=False)
    free = 200 << 30
    assert b._page_memory(free) == int(free * 0.85)
    # (the buffer that is too small and the one that takes its place: 4 bytes a float, grown by half)
    assert a._page_memory(free) <= 0.85 * (free - 4 * (ROOM + ROOM * 3 // 2)) and a._page_memory(free) > 0.84 * free
    assert a._page_memory(1 << 30) == int((1 << 29) * 0.85)


@pytest.mark.parametrize("requests", [4, 2, 1, 0])
def test_evictions_of_many_long_requests_go_some_at_a_time(bounded_ops, model, monkeypatch, requests):
    """20 of 30 to 60 tokens stay, listed for each of the model's layers and kv heads, 4 bytes each."""
    from litinfer_amd.engine import engine as module
    layers, heads = CFG["num_hidden_layers"], CFG["num_key_value_heads"]
    monkeypatch.setattr(module, "EVICT_ROOM", requests * 4 * layers * heads * 20)
    lists = []
    select = ops.evict_select
    monkeypatch.setattr(ops, "evict_select", lambda *a: lists.append(a[-1].shape) or select(*a))
    eng, alone = engine(model, num_pages=100), engine(model, num_pages=100)
    names = [f"r{i}" for i in range(4)]
    for e in (eng, alone):
        for i, rid in enumerate(names):
            e.step([StepEntry(rid, text(30 + 10 * i, i), [])])
    assert eng.evict(names, 20) == [20] * 4
    assert [shape[1] for shape in lists] == [max(1, requests)] * (4 // max(1, requests))
    for rid in names:
        alone.evict([rid], 20)
    eng.cache.check_invariants()
    for rid in names:
        step = [StepEntry(rid, [7], [0])]
        assert torch.equal(eng.step(step), alone.step(step))
