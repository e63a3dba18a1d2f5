"""What the backward of relative_attention takes the workspace to hold is what the forward wrote there, whatever becomes of the
saved tensors in between, without a GPU: the library's calls are replaced by a record of their arguments."""
import pytest
import torch

import fast_ops_b200._lib as L
from fast_ops_b200.flash_attention import relative

B, H, M, N, D = 2, 3, 4, 40, 8


class Recorder:
    def __init__(self, real):
        self.fo_rel_attn_workspace = real.fo_rel_attn_workspace

    @staticmethod
    def bias(args):
        """Whether there is one, its strides and its type (the last arguments: ..., p, seed, offset, device, stream)."""
        ptr, strides, code = args[-8:-5]
        return ptr is not None, None if strides is None else list(strides), code

    def fo_rel_attn_fwd(self, *args):
        self.forward_bias = self.bias(args)
        return 0

    def fo_rel_attn_bwd(self, *args):
        self.backward_bias = self.bias(args)
        return 0


def saved_elsewhere():
    """As torch.autograd.graph.save_on_cpu does: the tensors come back dense."""
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t)


@pytest.mark.parametrize("name,bias", [
    ("none", None),
    ("one row", torch.zeros(1, 1, 1, N)),
    ("one row expanded", torch.zeros(1, 1, 1, N).expand(B, H, 1, N)),
    ("heads expanded", torch.zeros(B, 1, 1, N).expand(B, H, 1, N)),
    ("batch expanded", torch.zeros(1, H, 1, N).expand(B, H, 1, N)),
    ("strided", torch.zeros(B, H, 1, 2 * N)[..., ::2]),
    ("each its own", torch.zeros(B, H, 1, N)),
])
@pytest.mark.parametrize("elsewhere", [False, True])
def test_the_backward_reads_the_rows_that_the_forward_wrote(name, bias, elsewhere, monkeypatch):
    rec = Recorder(L.load())
    monkeypatch.setattr(relative._lib, "load", lambda: rec)
    monkeypatch.setattr(relative._lib, "check", lambda rc: None)
    monkeypatch.setattr(relative._lib, "current_stream_ptr", lambda index: 0)
    prepare = relative._prepare_bias

    class OnDevice(torch.Tensor):
        is_cuda = True

    monkeypatch.setattr(relative, "_prepare_bias", lambda b, *args: prepare(b.as_subclass(OnDevice), *args))
    q, k, v = (torch.zeros(B, H, s, D, dtype=torch.bfloat16, requires_grad=True) for s in (M, N, N))
    table = torch.zeros(32, H)
    call = object.__new__(relative._Call)
    call.B, call.H, call.M, call.N, call.D = B, H, M, N, D
    call.code, call.device, call.index, call.table_code, call.num_buckets = L.FO_BF16, q.device, 0, L.FO_F32, 32
    call.key = (32, 128, True)
    call.starts, call.n_starts = relative._starts_array(*call.key)
    call.bidirectional, call.offset, call.causal, call.scale, call.dropout_p, call.rng = 1, 0, 0, 0.125, 0.0, (0, 0)
    if elsewhere:
        with saved_elsewhere():
            O = relative._RelativeAttentionFunction.apply(q, k, v, table, call, bias, False)
    else:
        O = relative._RelativeAttentionFunction.apply(q, k, v, table, call, bias, False)
    torch.autograd.grad(O, (q, k, v), torch.zeros_like(O))
    assert rec.forward_bias[0] == (bias is not None)
    assert rec.backward_bias == rec.forward_bias
