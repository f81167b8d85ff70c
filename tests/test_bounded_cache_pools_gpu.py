"""attention_mass where its single tokens' scores take more room than a launch has: several launches that use it one after the other."""
import pytest
import torch

import bounded_cache_cases as cases
from litinfer_amd.engine.workspace import Workspace
from litinfer_amd.kernels import ops
from test_bounded_cache_gpu import mass_inputs, mass_tolerance

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def widened(meta, blocks):
    """The same batch in tables of `blocks` pages."""
    meta.block_table = torch.nn.functional.pad(meta.block_table, (0, blocks - meta.max_blocks), value=-1).contiguous()
    meta.max_blocks = blocks
    return meta


def one_by_one(qkv, mass, k, meta, nh, nkv, dh, page_size, scale):
    """The batch's requests in calls of their own: these fit the room."""
    out = mass.clone()
    for r in range(meta.num_segments):
        part = cases.batch([(1, int(meta.host_ctx_len[r]))], page_size, DEV)[0]
        part.block_table, part.max_blocks = meta.block_table[r:r + 1].contiguous(), meta.max_blocks
        ops.attention_mass(qkv[r:r + 1], out, k, part, nh, nkv, dh, page_size, scale)
    return out


@pytest.mark.parametrize("segs,nh,nkv", [([(1, 50000)] * 4 + [(1, 30001)], 320, 1), ([(1, 2600 + 17 * i) for i in range(70)], 320, 1)])
def test_mass_of_batches_in_several_launches(segs, nh, nkv):
    """Named requests, and more than are named: 2^26 floats hold some 200,000 keys of 320 heads."""
    dh, scale, ws = 64, 0.125, Workspace(DEV)
    assert sum(-(-c // 64) * 66 * nh for _, c in segs) > 1 << 26
    qkv, mass, k, meta = mass_inputs(segs, nh, nkv, dh, 16, torch.bfloat16)
    start = mass.clone()
    want = one_by_one(qkv, mass, k, meta, nh, nkv, dh, 16, scale)
    for _ in range(2):
        mass.copy_(start)
        ops.attention_mass(qkv, mass, k, meta, nh, nkv, dh, 16, scale, ws=ws)
        assert torch.equal(mass, want)
    plain = cases.plain_mass(qkv, start, k, meta, nh, nkv, dh, 16, scale)
    assert torch.allclose(mass.cpu().double(), plain, rtol=mass_tolerance(qkv, k, meta, nh, nkv, dh, scale), atol=1e-30)


def test_mass_of_a_recording_whose_tables_take_more_than_the_room():
    """64 requests of 40 heads in tables of 2,048 pages: a launch has room for 49 of them."""
    nh, nkv, dh, scale, ws = 40, 8, 64, 0.125, Workspace(DEV)
    qkv, mass, k, meta = mass_inputs([(1, 2100 + 41 * i) for i in range(64)], nh, nkv, dh, 16, torch.bfloat16)
    widened(meta, 2048)
    start = mass.clone()
    want = one_by_one(qkv, mass, k, meta, nh, nkv, dh, 16, scale)
    meta.padded = True
    ops.attention_mass(qkv, mass, k, meta, nh, nkv, dh, 16, scale, ws=ws)
    assert torch.equal(mass, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_mass(qkv, mass, k, meta, nh, nkv, dh, 16, scale, ws=ws)
    for _ in range(3):
        mass.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mass, want)
        torch.randn(1000, device=DEV).sum().item()
    assert ws.buffer("evict.mass", (1,), torch.float32).untyped_storage().size() <= 4 << 26
