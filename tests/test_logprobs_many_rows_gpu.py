"""token_logprobs of more rows than one launch has threads for."""
import pytest
import torch

from litinfer_amd.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = 2.0 ** -24


def test_logprobs_of_more_rows_than_a_launch_takes():
    """2^23 rows of 512 threads are 2^32; the rows' values against 64 bits: three roundings of the two differences and the logarithm, and eight
    of a sum of three shares, of whose weight none is above one."""
    n = (1 << 23) + 1025
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(n, 3, generator=g, device=DEV)
    ids = torch.randint(0, 3, (n,), generator=g, device=DEV, dtype=torch.int32)
    lp, ent = torch.full((n,), 9.0, device=DEV), torch.full((n,), 9.0, device=DEV)
    ti, tl = torch.full((n, 2), 9, dtype=torch.int32, device=DEV), torch.full((n, 2), 9.0, device=DEV)
    ops.token_logprobs(x, ids, lp, ent, ti, tl)
    y = torch.log_softmax(x.double(), 1)
    want = y.gather(1, ids.long()[:, None])[:, 0]
    assert bool(((lp.double() - want).abs() <= (80 + 3 * want.abs()) * HALF).all())
    entropy = -(y.exp() * y).sum(1)
    assert bool(((ent.double() - entropy).abs() <= 160 * HALF * (1 + entropy)).all())
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(ti.long(), order)
    top = y.gather(1, order)
    assert bool(((tl.double() - top).abs() <= (80 + 3 * top.abs()) * HALF).all())
