"""Forward-mode derivatives are refused, not dropped.  The device calls are replaced by zeros of the right shape."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from fast_ops_b200.flash_attention import flash_attention, flash_attention_bshd, relative


class Call:
    """Stands in for the checked arguments of a relative attention call."""

    def __init__(self, *_):
        pass

    def forward(self, Q, K, V, table, bias, lse):
        return torch.zeros(Q.shape), torch.zeros(Q.shape[:3]) if lse else None, None


def zeros(Q, K, V, *args, **kwargs):
    return (torch.zeros(Q.shape), torch.zeros(Q.shape[:3])) if kwargs.get("return_lse") or (len(args) > 3 and args[3]) else torch.zeros(Q.shape)


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(relative, "_Call", Call)
    monkeypatch.setattr(flash_attention, "_forward", zeros)
    monkeypatch.setattr(flash_attention_bshd, "_forward", zeros)
    for module in (flash_attention, flash_attention_bshd):
        monkeypatch.setattr(module, "next_dropout_rng", lambda device, count: (0, 0))


CALLS = {
    "relative": lambda q, k, v, t: relative.relative_attention(q, k, v, t),
    "relative with LSE": lambda q, k, v, t: relative.relative_attention(q, k, v, t, return_lse=True),
    "plain": lambda q, k, v, t: flash_attention.multi_head_attention(q, k, v),
    "causal": lambda q, k, v, t: flash_attention.multi_head_attention(q, k, v, causal=True),
    "dropout and LSE": lambda q, k, v, t: flash_attention.multi_head_attention(q, k, v, dropout_p=0.1, return_lse=True),
    "bshd": lambda q, k, v, t: flash_attention_bshd.flash_attn_bshd(q, k, v),
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(name, which, grad, on_cpu):
    if which == 3 and not name.startswith("relative"):
        pytest.skip("no table")
    tensors = [torch.zeros(1, 2, 4, 8) for _ in range(3)] + [torch.zeros(32, 2)]
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        tensors[which] = fwd.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with pytest.raises(RuntimeError):
            CALLS[name](*tensors)


@pytest.mark.parametrize("name", CALLS)
def test_calls_without_a_tangent_go_on(name, on_cpu):
    tensors = [torch.zeros(1, 2, 4, 8) for _ in range(3)] + [torch.zeros(32, 2)]
    with fwd.dual_level():
        out = CALLS[name](*tensors)
    assert not (out[0] if isinstance(out, tuple) else out).requires_grad
    out = CALLS[name](*tensors)
    assert (out[0] if isinstance(out, tuple) else out).shape == tensors[0].shape
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: CALLS[name](q, *tensors[1:]), (tensors[0],), (tensors[0],))
