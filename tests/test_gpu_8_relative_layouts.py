"""relative_attention's gradients for layouts that a training step can meet: the same as for dense copies, bit for bit where
the sums have a fixed order (dQ is summed by atomic adds)."""
import pytest
import torch

from fast_ops_b200.flash_attention import multi_head_attention, relative_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def same(got, want):
    for i in (1, 2, 3):
        assert torch.equal(got[i], want[i]), i
    assert torch.allclose(got[0].float(), want[0].float(), rtol=2.0**-7, atol=1e-6)


def inputs(B, H, M, N, D, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.empty(s, dtype=BF, device="cuda").normal_(generator=gen)  # noqa: E731
    return r(B, H, M, D), r(B, H, N, D), r(B, H, N, D), r(32, H), r(B, H, M, D)


@pytest.mark.parametrize("M", [1, 100])
@pytest.mark.parametrize("at", [1, 4])
def test_an_output_gradient_that_begins_between_aligned_addresses(M, at, cuda_device):
    Q, K, V, table, dO = inputs(2, 3, M, 130, 64)
    leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]
    O = relative_attention(*leaves)
    flat = torch.zeros(dO.numel() + 8, dtype=BF, device="cuda")
    g = flat[at:at + dO.numel()].view(dO.shape)
    g.copy_(dO)
    assert g.is_contiguous() and g.data_ptr() % 16
    same(torch.autograd.grad(O, leaves, g, retain_graph=True), torch.autograd.grad(O, leaves, dO))


@pytest.mark.parametrize("M,N", [(1, 130), (70, 1), (1, 1)])
def test_rows_of_stride_one_where_there_is_one_row(M, N, cuda_device):
    """(B, H, D, 1) tensors transposed: the gradients of Q or of K and V get the same strides."""
    Q, K, V, table, dO = inputs(2, 3, M, N, 64)
    want_leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]
    want = torch.autograd.grad(relative_attention(*want_leaves), want_leaves, dO)
    column = lambda t: t.clone().view(2, 3, 64, 1).transpose(2, 3) if t.shape[2] == 1 else t.clone()  # noqa: E731
    leaves = [column(t).requires_grad_() for t in (Q, K, V)] + [table.clone().requires_grad_()]
    assert any(t.stride(2) == 1 for t in leaves[:3])
    same(torch.autograd.grad(relative_attention(*leaves), leaves, dO), want)
    plain = torch.autograd.grad(multi_head_attention(*leaves[:3]), leaves[:3], dO)
    dense = torch.autograd.grad(multi_head_attention(*want_leaves[:3]), want_leaves[:3], dO)
    same(plain + (table,), dense + (table,))
