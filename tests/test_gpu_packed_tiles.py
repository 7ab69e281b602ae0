"""packed_attention where its tiles end: rows behind the last next to infinities."""
import math

import pytest
import torch

from test_gpu_packed_attention import attend, tensors

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def run(q, k, v, g, ptr, kv_ptr=None, **kw):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    y = attend(*leaves, ptr, kv_ptr, **kw)
    return [y.detach(), *torch.autograd.grad(y, leaves, g)]


# rows of a key's tile: below, at and above 16, 32 and 64 rows of queries and heads
@pytest.mark.parametrize("t,d", [(torch.float32, 8), (torch.float32, 16), (torch.float32, 40),
                                 (torch.bfloat16, 16), (torch.bfloat16, 64), (torch.bfloat16, 128)], ids=str)
@pytest.mark.parametrize("h,hk", [(1, 1), (6, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_a_key_of_probability_zero(causal, h, hk, t, d):
    """A key with -inf in a dimension where all queries are positive: its probability is 0 and
    so are dk and dv, at every number of rows, as with a finite value far enough down."""
    for n in (2, 5, 11, 16, 22, 31, 32, 33, 43, 64, 65, 100, 700):
        q, k, v = tensors(n, n, h, hk, d, t, seed=n)
        g = torch.randn(n, h, d, device=DEV).to(t)
        q[..., 0] = q[..., 0].abs() + 0.5
        ptr = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        for at in {1, n // 2, n - 1} - {0}:
            got = []
            for low in (-1e30, -math.inf):
                k[at, :, 0] = low
                got.append(run(q, k, v, g, ptr, causal=causal))
            k[at, :, 0] = 1.0
            for name, j in (("y", 0), ("dk", 2), ("dv", 3)):
                assert bool(got[1][j].isfinite().all()), (name, n, at)
                assert torch.equal(got[0][j], got[1][j]), (name, n, at)
            assert not got[1][2][at].any() and not got[1][3][at].any()
            # dq: 0 times -inf in that dimension alone
            assert torch.equal(got[0][1][..., 1:], got[1][1][..., 1:])
