"""Sizes beyond what the kernels' 32-bit loops and arguments hold are refused, before anything is launched: by the Python entry, on tensors
that have a shape and no memory, and by the library itself."""
import pytest
import torch

import bounded_cache_cases as cases
from litinfer_amd.kernels import ops
from test_bounded_cache_cpu import no_gpu  # noqa: F401 (a fixture)

REFUSED = 2                            # the library's code for sizes that it does not take


def f32(*shape):
    return torch.empty(shape, dtype=torch.float32, device="meta")


def i32(*shape):
    return torch.empty(shape, dtype=torch.int32, device="meta")


MANY = (1 << 30) + 1


@pytest.mark.parametrize("change", [dict(out=i32(1, 1, 1, MANY)), dict(out=i32(1, 1, 1, (1 << 31) - 1)), dict(out=i32(1, 1, 1, (1 << 32) + 4)),
                                    dict(block_table=i32(1, (1 << 26) + 1)), dict(block_table=i32(1, (1 << 32) + 4)),
                                    dict(mass=f32(1, 1 << 31, 1, 16, 1)), dict(mass=f32(1, (1 << 32) + 9, 1, 16, 1))])
def test_evict_select_refuses(no_gpu, change):  # noqa: F811
    call = dict(mass=f32(1, 9, 1, 16, 1), block_table=i32(1, 4), lens=i32(1), keep=i32(1), first=1, recent=2, out=i32(1, 1, 1, 8))
    with pytest.raises(ValueError, match="evict_select: .*2.3[01]"):
        ops.evict_select(**{**call, **change})


@pytest.mark.parametrize("change", [dict(kept=i32(1, 1, 1, MANY)), dict(kept=i32(1, 1, 1, (1 << 32) + 4)), dict(block_table=i32(1, (1 << 26) + 1)),
                                    dict(tensors=[f32(1, 1 << 27, 1, 16, 4)]), dict(tensors=[f32(1, (1 << 32) + 9, 1, 16, 4)])])
def test_cache_compact_refuses(no_gpu, change):  # noqa: F811
    call = dict(tensors=[f32(1, 9, 1, 16, 4)], block_table=i32(1, 4), kept=i32(1, 1, 1, 8))
    with pytest.raises(ValueError, match="cache_compact: .*2.3[01]"):
        ops.cache_compact(**{**call, **change})


def test_attention_mass_refuses(no_gpu):  # noqa: F811
    def call(pages=None, blocks=None, stride=None):
        meta, held = cases.batch([(1, 3), (1, 80)], 16, "cpu")
        pages = held if pages is None else pages
        if blocks:
            meta.block_table, meta.max_blocks = i32(2, blocks), blocks
        qkv = f32(2, 64) if stride is None else torch.empty_strided((2, 64), (stride, 1), device="meta")
        ops.attention_mass(qkv, f32(pages, 2, 16, 1), f32(pages, 2, 16, 8), meta, 4, 2, 8, 16, 1.0)
    for change in (dict(pages=1 << 26), dict(pages=(1 << 32) + 9), dict(blocks=(1 << 26) + 1), dict(stride=1 << 31), dict(stride=(1 << 32) + 64)):
        with pytest.raises(ValueError, match="attention_mass: .*2.3[01]"):
            call(**change)


@pytest.mark.parametrize("max_blocks,page_size,K", [((1 << 26) + 1, 16, 8), (1 << 30, 2, 8), (4, 16, MANY), (4, 16, (1 << 31) - 1)])
def test_the_library_refuses(max_blocks, page_size, K):
    assert ops._fn("evict", "li_evict_select")(0, 0, max_blocks, 0, 0, 1, 0, 0, 0, K, 1, 1, page_size, 9, 0) == REFUSED
    assert ops._fn("evict", "li_cache_compact")(0, 0, 1, 0, max_blocks, 0, K, 1, 1, 1, page_size, 9, 0) == REFUSED
    if K == 8:
        one = (ops.c_int * 1)(1)
        at = ops.ctypes.addressof(one)
        assert ops._fn("evict", "li_attention_mass")(0, 64, 0, 0, 0, 0, max_blocks, 0, 0, 0, at, at, at, 1, 1, 0, 4, 2, 8, page_size, 9, 1.0, 1, at, 1 << 20, 0) == REFUSED


@pytest.mark.parametrize("rows", [MANY, (1 << 31) - 1, (1 << 32) + 5])
def test_token_logprobs_refuses(no_gpu, rows):  # noqa: F811
    with pytest.raises(ValueError, match="token_logprobs: .* rows .*2.30"):
        ops.token_logprobs(f32(rows, 2), i32(rows), f32(rows), f32(rows))
    if rows < 1 << 31:
        one = (ops.c_int * 1)(1)
        assert ops._fn("logprobs", "li_token_logprobs")(0, 2, 0, rows, 2, 0, 0, 0, 0, 0, ops.ctypes.addressof(one), 0) == REFUSED


def test_the_limits_that_python_names_are_the_library_s():
    """One more is refused by the library; the limits themselves are taken by the tests on the GPU (32 alternatives) or by their arithmetic."""
    one = (ops.c_int * 1)(1)
    call = ops._fn("logprobs", "li_token_logprobs")
    for v, top in ((ops.LOGPROBS_MAX_VOCAB + 1, 0), (99, ops.LOGPROBS_MAX_TOP + 1)):
        assert call(0, 1 << 22, 0, 1, v, top, 0, 0, 0, 0, ops.ctypes.addressof(one), 0) == REFUSED
