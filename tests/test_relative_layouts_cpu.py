"""What the backward of relative_attention hands to the library for gradients and inputs of unusual layouts, without a GPU:
the library's call is replaced by a record of its arguments."""
import ctypes

import pytest
import torch

import fast_ops_b200._lib as L
from fast_ops_b200.flash_attention import relative

BF = torch.bfloat16


class Recorder:
    def __init__(self):
        self.args = None

    def fo_rel_attn_bwd(self, *args):
        self.args = args
        B, H, M, _, D = args[13:18]
        self.dO = tensor_at(args[4], (B, H, M, D), list(args[22]))
        return 0


def backward(monkeypatch, dO, Q, K, V):
    """(dQ, dK, dV), and the record of the library's call."""
    rec = Recorder()
    monkeypatch.setattr(relative._lib, "load", lambda: rec)
    monkeypatch.setattr(relative._lib, "check", lambda rc: None)
    monkeypatch.setattr(relative._lib, "current_stream_ptr", lambda index: 0)
    call = object.__new__(relative._Call)
    call.B, call.H, call.M, call.D = Q.shape
    call.N, call.device, call.code, call.causal, call.scale = K.shape[2], Q.device, L.FO_BF16, 0, 0.125
    call.table_code, call.starts, call.n_starts, call.bidirectional, call.offset = L.FO_F32, None, 0, 1, 0
    call.dropout_p, call.rng, call.index, call.bias_args = 0.0, (0, 0), 0, (None, None, L.FO_F32)
    O = torch.zeros(Q.shape, dtype=BF)
    return call.backward(dO, Q, K, V, O, torch.zeros(Q.shape[:3]), torch.zeros(16), None)[:3], rec


def tensor_at(ptr, shape, strides):
    """The bf16 values that a pointer and (batch, head, row) strides stand for."""
    out = torch.empty(shape, dtype=torch.int16)
    for b in range(shape[0]):
        for h in range(shape[1]):
            for s in range(shape[2]):
                row = (ctypes.c_int16 * shape[3]).from_address(ptr + 2 * (b * strides[0] + h * strides[1] + s * strides[2]))
                out[b, h, s] = torch.tensor(list(row), dtype=torch.int16)
    return out.view(BF)


def gradients(shape):
    B, H, M, D = shape
    whole = torch.randn(B, H, M, D).bfloat16()
    yield "dense", whole
    flat = torch.zeros(whole.numel() + 8, dtype=BF)
    for at in (1, 4):
        flat[at:at + whole.numel()] = whole.reshape(-1)
        yield f"dense, {2 * at} bytes behind an aligned address", flat[at:at + whole.numel()].view(shape)
    yield "cut", torch.randn(B, H, M, D + 1).bfloat16()[..., 1:]
    yield "expanded over the batch", whole[:1].expand(shape)
    yield "a number", torch.ones((), dtype=BF).expand(shape)
    yield "transposed", torch.randn(B, M, H, D).bfloat16().transpose(1, 2)


@pytest.mark.parametrize("shape", [(2, 3, 5, 8), (2, 3, 1, 16), (1, 1, 1, 8)])
def test_output_gradients_reach_the_library_in_a_layout_that_it_takes(shape, monkeypatch):
    Q, K = torch.zeros(shape, dtype=BF), torch.zeros(*shape[:2], 4, shape[3], dtype=BF)
    for name, dO in gradients(shape):
        _, record = backward(monkeypatch, dO, Q, K, K)
        ptr, strides = record.args[4], list(record.args[22])
        assert ptr % 16 == 0, name
        for extent, stride in zip(shape, strides):
            assert extent == 1 or (stride > 0 and stride % 8 == 0), name
        assert torch.equal(record.dO, dO), name
        monkeypatch.undo()


@pytest.mark.parametrize("entry", ["fo_rel_attn_bwd", "fo_flash_attn_bwd"])
def test_a_dimension_of_extent_1_may_have_any_stride(entry):
    """A (B, H, D, 1) tensor transposed to (B, H, 1, D) has row stride 1, and so has a gradient made like it.  (dv's strides
    are wrong on purpose: they are checked behind the others, and before any CUDA call.)"""
    lib = L.load()
    i3 = ctypes.c_int64 * 3
    one, rows, wrong = i3(2 * 64, 64, 1), i3(8 * 64 * 2, 8 * 64, 64), i3(8 * 64 * 2, 8 * 64, 63)

    def call(o, dq, dk, dv, H=2, Sq=1):
        if entry == "fo_rel_attn_bwd":
            starts = (ctypes.c_int * 2)(0, 1)
            lib.fo_rel_attn_bwd(*([16] * 9), None, 16, 16, None, 1, H, Sq, 8, 64, one, rows, rows, o, one, dq, dk, dv,
                                L.FO_BF16, 0, 0.125, L.FO_F32, starts, 2, 1, 0, 16, None, None, L.FO_F32, 0.0, 0, 0, 0, None)
        else:
            lib.fo_flash_attn_bwd(*([16] * 11), 1, H, Sq, 8, 64, one, rows, rows, o, one, dq, dk, dv, L.FO_BF16, 0, 0.125, 0, None)
        return lib.fo_last_error()

    assert call(one, one, rows, wrong).startswith(b"dv: strides")
    assert call(i3(3, 64, 1), i3(5, 64, 7), i3(7, 8 * 64, 64), wrong).startswith(b"dv: strides")  # a batch of one too
    assert call(one, one, rows, wrong, Sq=2).startswith(b"o: strides")
    assert call(rows, one, rows, wrong, Sq=2).startswith(b"dq: strides")
    assert call(one, one, wrong, rows).startswith(b"dk: strides")
    assert call(one, i3(128, 4, 1), rows, wrong, H=1).startswith(b"dv: strides")
