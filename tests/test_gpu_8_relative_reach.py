"""Buckets that reach far: forward, gradients and the table's gradient against 64 bits."""
import pytest
import torch

import fast_ops_b200._lib as L
from fast_ops_b200.flash_attention import relative_attention
from table_gradient_bound import expected
from test_gpu_8_relative_attention import close, formula

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype,M,N,offset,bid,md", [
    (128, torch.bfloat16, 1000, 1000, 0, True, 4000), (128, torch.float16, 300, 2000, 1700, False, 3000),
    (96, torch.bfloat16, 1100, 1200, 0, True, 4000), (64, torch.bfloat16, 2100, 2100, 0, True, 8000),
    (64, torch.float16, 700, 4200, 3500, False, 8000)])
@pytest.mark.parametrize("padded", [False, True])
def test_buckets_that_reach_past_shared_memory(D, dtype, M, N, offset, bid, md, padded, cuda_device):
    """The bias vector of these does not fit beside two CTAs on an SM: the forward takes the kernel that reads it from the
    first-level cache, by its own rule."""
    B, H = 1, 2
    gen = torch.Generator(device="cuda").manual_seed(N)
    r = lambda *s: torch.empty(s, dtype=dtype, device="cuda").normal_(generator=gen)  # noqa: E731
    Q, K, V, dO = r(B, H, M, D), r(B, H, N, D), r(B, H, N, D), r(B, H, M, D)
    table = torch.empty(32, H, device="cuda").normal_(generator=gen)
    bias = None
    if padded:
        bias = torch.zeros(B, 1, 1, N, device="cuda")
        bias[..., N - 333:] = -float("inf")
    kw = dict(max_distance=md, bidirectional=bid, causal=not bid, bias=bias)
    leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]
    O, lse = relative_attention(*leaves, query_offset=offset, return_lse=True, **kw)
    got = (O.detach(), lse) + torch.autograd.grad(O, leaves, dO)
    want, tol = formula(Q, K, V, table, dO, offset=offset, **kw)
    close("O", got[0], want["O"], tol["O"])
    assert (lse.double() - want["LSE"]).abs().max().item() <= 2e-5
    for name, x in zip(("dQ", "dK", "dV"), got[2:5]):
        close(name, x, want[name], tol[name])
    want_t, bound = expected(Q, K, V, table, dO, offset=offset, **kw)
    assert ((got[5].double() - want_t).norm(dim=0) <= bound.norm(dim=0)).all()
    torch.cuda.synchronize()
    assert L.device_status(0) == 0
