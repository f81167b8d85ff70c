"""What the operators around a cache of bounded length and token_logprobs refuse: before anything is launched."""
import pytest
import torch

import bounded_cache_cases as cases
from litinfer_amd.kernels import ops


@pytest.fixture
def no_gpu(monkeypatch):
    """The argument checks alone: tensors may lie on the host, and nothing may be launched."""
    def launched(*a, **k):
        raise AssertionError("a call that has to be refused was launched")
    monkeypatch.setattr(ops, "_here", lambda what, *ts: None)
    monkeypatch.setattr(ops, "_run", launched)


def f32(*shape):
    return torch.zeros(shape)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="not on the GPU"):
        ops.token_logprobs(f32(2, 9), i32(2), f32(2), f32(2))
    with pytest.raises(RuntimeError, match="not on the GPU"):
        ops.evict_select(f32(1, 4, 2, 16, 1), i32(1, 4), i32(1), i32(1), 0, 0, i32(1, 1, 2, 8))
    with pytest.raises(RuntimeError, match="not on the GPU"):
        ops.cache_compact([f32(1, 4, 2, 16, 8)], i32(1, 4), i32(1, 1, 2, 8))
    meta, pages = cases.batch([(1, 3)], 16, "cpu")
    with pytest.raises(RuntimeError, match="not on the GPU"):
        ops.attention_mass(f32(1, 4 * 8 * 2), f32(pages, 2, 16, 1), f32(pages, 2, 16, 8), meta, 4, 2, 8, 16, 1.0)


@pytest.mark.parametrize("change", [dict(logits=f32(2, 9).double()), dict(logits=f32(9, 2).t()), dict(logits=f32(2, 9)[:, ::2]), dict(ids=i32(3)), dict(ids=i32(2).long()),
                                    dict(ids=i32(2, 1)), dict(logprobs=f32(3)), dict(entropy=f32(2).double()), dict(top_ids=i32(2, 3)), dict(top_logprobs=f32(2, 3)),
                                    dict(top_ids=i32(2, 3), top_logprobs=f32(2, 4)), dict(top_ids=i32(2, 10), top_logprobs=f32(2, 10)),
                                    dict(logits=f32(2, 99), top_ids=i32(2, 33), top_logprobs=f32(2, 33)), dict(logits=f32(2, (1 << 20) + 1)),
                                    dict(top_ids=i32(2, 3).long(), top_logprobs=f32(2, 3)), dict(logits=f32(2, 0))])
def test_token_logprobs_refuses(no_gpu, change):
    call = dict(logits=f32(2, 9), ids=i32(2), logprobs=f32(2), entropy=f32(2), **{})
    with pytest.raises(ValueError, match="token_logprobs"):
        ops.token_logprobs(**{**call, **change})


def test_no_rows_are_no_call(no_gpu):
    ops.token_logprobs(f32(0, 9), i32(0), f32(0), f32(0))


@pytest.mark.parametrize("change", [dict(mass=f32(9, 2, 16, 1).double()), dict(mass=f32(9, 2, 16)), dict(k=f32(9, 2, 16, 6)), dict(k=f32(9, 2, 16, 8).bfloat16()),
                                    dict(nh=3), dict(dh=7), dict(dh=258), dict(qkv=f32(41, 31)), dict(qkv=f32(40, 64)), dict(page_size=8), dict(k=f32(9, 2, 8, 16).transpose(2, 3))])
def test_attention_mass_refuses(no_gpu, change):
    meta, pages = cases.batch([(1, 3), (40, 80)], 16, "cpu")
    call = dict(qkv=f32(41, 64), mass=f32(pages, 2, 16, 1), k=f32(pages, 2, 16, 8), meta=meta, nh=4, nkv=2, dh=8, page_size=16, scale=1.0)
    assert pages == 9
    with pytest.raises(ValueError):
        ops.attention_mass(**{**call, **change})


def test_attention_mass_refuses_a_batch_that_does_not_fit(no_gpu):
    for name, value in (("block_table", i32(2, 3)), ("block_table", i32(2, 6).long()), ("max_ctx_len", 97), ("q_len", i32(3)), ("ctx_len", i32(2).long()), ("num_tokens", 40)):
        meta, pages = cases.batch([(1, 3), (40, 80)], 16, "cpu")
        setattr(meta, name, value)
        with pytest.raises(ValueError, match="attention_mass"):
            ops.attention_mass(f32(41, 64), f32(pages, 2, 16, 1), f32(pages, 2, 16, 8), meta, 4, 2, 8, 16, 1.0)


@pytest.mark.parametrize("change", [dict(mass=f32(3, 9, 2, 16)), dict(mass=f32(3, 9, 2, 16, 2)), dict(mass=f32(3, 9, 2, 16, 1).double()), dict(block_table=i32(5, 4)),
                                    dict(block_table=i32(4, 4).long()), dict(lens=i32(5)), dict(keep=i32(3)), dict(first=-1), dict(recent=-2), dict(out=i32(3, 4, 2, 8).long()),
                                    dict(out=i32(3, 4, 3, 8)), dict(out=i32(2, 4, 2, 8)), dict(mass=f32(3, 9, 16, 2, 1).transpose(2, 3)), dict(block_table=i32(4, 0))])
def test_evict_select_refuses(no_gpu, change):
    call = dict(mass=f32(3, 9, 2, 16, 1), block_table=i32(4, 4), lens=i32(4), keep=i32(4), first=1, recent=2, out=i32(3, 4, 2, 8))
    with pytest.raises(ValueError, match="evict_select"):
        ops.evict_select(**{**call, **change})


@pytest.mark.parametrize("change", [dict(tensors=[]), dict(tensors=[f32(3, 9, 2, 16, 4)] * 5), dict(tensors=[f32(3, 9, 2, 16, 4), f32(3, 8, 2, 16, 4)]),
                                    dict(tensors=[f32(3, 9, 2, 16, 3).bfloat16()]), dict(tensors=[f32(2, 9, 2, 16, 4)]), dict(tensors=[f32(3, 9, 3, 16, 4)]),
                                    dict(tensors=[f32(3, 9, 2, 4, 16).transpose(3, 4)]), dict(block_table=i32(5, 4)), dict(kept=i32(3, 4, 2, 8).long()), dict(kept=i32(3, 4, 2))])
def test_cache_compact_refuses(no_gpu, change):
    call = dict(tensors=[f32(3, 9, 2, 16, 4)], block_table=i32(4, 4), kept=i32(3, 4, 2, 8))
    with pytest.raises(ValueError, match="cache_compact"):
        ops.cache_compact(**{**call, **change})
