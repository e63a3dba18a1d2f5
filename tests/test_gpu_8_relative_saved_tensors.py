"""relative_attention where its saved tensors are kept elsewhere between forward and backward: on the host, in a checkpoint,
or packed so that they come back with other strides."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from fast_ops_b200.flash_attention import relative_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
B, H, M, N, D = 2, 3, 200, 333, 64


def inputs():
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.empty(s, dtype=BF, device="cuda").normal_(generator=gen)  # noqa: E731
    return r(B, H, M, D), r(B, H, N, D), r(B, H, N, D), r(32, H), r(B, H, M, D)


def biases():
    row = torch.zeros(1, 1, 1, N, device="cuda")
    row[..., 300:] = -float("inf")
    heads = torch.randn(1, H, 1, N, device="cuda")
    yield None
    yield row.expand(B, H, 1, N)
    yield heads.expand(B, H, 1, N)
    yield torch.randn(B, 1, 1, N, device="cuda").expand(B, H, 1, N)
    yield torch.randn(B, H, 1, 2 * N, device="cuda")[..., ::2]


def same(got, want):
    for i in (1, 2, 3):
        assert torch.equal(got[i], want[i]), i
    assert torch.allclose(got[0].float(), want[0].float(), rtol=2.0**-7, atol=1e-6)  # dQ is summed by atomic adds


@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("how", ["on the host", "packed densely"])
def test_saved_tensors_that_come_back_dense(how, p, cuda_device):
    Q, K, V, table, dO = inputs()
    rng = (3, 4) if p else None
    hooks = torch.autograd.graph.save_on_cpu() if how == "on the host" else torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t)
    for bias in biases():
        leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]
        want = torch.autograd.grad(relative_attention(*leaves, bias=bias, dropout_p=p, rng=rng), leaves, dO)
        with hooks:
            O = relative_attention(*leaves, bias=bias, dropout_p=p, rng=rng)
        same(torch.autograd.grad(O, leaves, dO), want)


def test_inputs_with_strides_and_shared_heads_on_the_host(cuda_device):
    Q, K, V, table, dO = inputs()
    q = Q.transpose(1, 2).contiguous().requires_grad_()
    k, v = (t[:, :1].clone().requires_grad_() for t in (K, V))
    t = table.clone().requires_grad_()
    leaves = (q, k, v, t)

    def run():
        return relative_attention(q.transpose(1, 2), k.expand(B, H, N, D), v.expand(B, H, N, D), t)

    want = torch.autograd.grad(run(), leaves, dO)
    with torch.autograd.graph.save_on_cpu():
        O = run()
    same(torch.autograd.grad(O, leaves, dO), want)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_checkpointing(reentrant, p, cuda_device):
    """The forward is run again in the backward, with the dropout mask of the first time."""
    Q, K, V, table, dO = inputs()
    bias = next(b for b in biases() if b is not None)
    leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]

    def run(*args):
        return relative_attention(*args, bias=bias, dropout_p=p)

    torch.cuda.manual_seed(5)
    want = torch.autograd.grad(run(*leaves), leaves, dO)
    torch.cuda.manual_seed(5)
    O = checkpoint(run, *leaves, use_reentrant=reentrant)
    O.backward(dO)
    same([t.grad for t in leaves], want)


def test_a_bias_changed_after_the_forward(cuda_device):
    """The gradients are those of the forward's bias."""
    Q, K, V, table, dO = inputs()
    bias = torch.randn(B, 1, 1, N, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]
    want = torch.autograd.grad(relative_attention(*leaves, bias=bias), leaves, dO)
    O = relative_attention(*leaves, bias=bias)
    bias.fill_(-float("inf"))
    same(torch.autograd.grad(O, leaves, dO), want)
