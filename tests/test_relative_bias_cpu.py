"""Buckets of the relative position bias, and what its entry points refuse, without a GPU."""
import ctypes
import math
from fractions import Fraction

import pytest
import torch

import fast_ops_b200._lib as L
from fast_ops_b200.flash_attention import relative_attention, relative_bucket_starts


def bucket_of(starts, n):
    return max(u for u, s in enumerate(starts) if s <= n)


@pytest.mark.parametrize("num_buckets,max_distance,bidirectional", [
    (32, 128, True), (32, 128, False), (64, 640, True), (16, 32, False), (4, 3, True), (2, 5, False), (6, 100_000, True),
    (512, 2000, True), (5, 3, False), (20, 11, False), (256, 100_000, False)])
def test_bucket_starts_follow_the_logarithm_exactly(num_buckets, max_distance, bidirectional):
    starts = relative_bucket_starts(num_buckets, max_distance, bidirectional)
    per_side = num_buckets // 2 if bidirectional else num_buckets
    exact = per_side // 2
    assert len(starts) == per_side and starts[:exact + 1] == tuple(range(exact + 1))
    assert all(a <= b for a, b in zip(starts, starts[1:])) and starts[-1] <= max_distance
    steps = per_side - exact
    for x, n in enumerate(starts[exact:]):
        # n is the smallest with (n / exact)^steps >= (max_distance / exact)^x
        bound = Fraction(max_distance, exact) ** x
        assert Fraction(n, exact) ** steps >= bound
        assert n == exact or Fraction(n - 1, exact) ** steps < bound


def test_buckets_by_the_usual_formula():
    """floor of the scaled logarithm, wherever its argument is not within 1e-9 of a border."""
    for num_buckets, max_distance, bidirectional in ((32, 128, True), (32, 128, False), (64, 640, True), (48, 1000, False)):
        starts = relative_bucket_starts(num_buckets, max_distance, bidirectional)
        exact, per_side = len(starts) // 2, len(starts)
        for n in range(2 * max_distance):
            if n < exact:
                want = n
            else:
                x = math.log(n / exact) / math.log(max_distance / exact) * (per_side - exact)
                if abs(x - round(x)) < 1e-9:
                    x = round(x)
                want = min(per_side - 1, exact + math.floor(x))
            assert bucket_of(starts, n) == want, (num_buckets, n)


@pytest.mark.parametrize("args", [(1, 128, False), (2, 128, True), (33, 128, True), (514, 5000, True), (257, 5000, False),
                                  (32, 8, True), (32, 0, False), (32, 2**29, True)])
def test_bucket_refusals(args):
    with pytest.raises(RuntimeError):
        relative_bucket_starts(*args)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        relative_attention(q, q, q, torch.zeros(32, 2))
    with pytest.raises(RuntimeError, match="tensors"):
        relative_attention(q, q, q, None)


def starts_array(*values):
    return (ctypes.c_int * len(values))(*values), len(values)


def forward_args(lib, **change):
    s = (ctypes.c_int64 * 3)(8 * 64 * 2, 8 * 64, 64)
    starts, n = starts_array(0, 1, 2, 5)
    a = dict(q=16, k=16, v=16, o=16, lse=None, B=1, H=2, Sq=8, Sk=8, D=64, qs=s, ks=s, vs=s, os=s, dtype=L.FO_BF16, causal=0,
             scale=0.125, table=16, ts=(ctypes.c_int64 * 2)(2, 1), table_dtype=L.FO_F32, starts=starts, n=n, two_sided=1,
             offset=0, workspace=16, bias=None, bs=None, bias_dtype=L.FO_F32, p=0.0, seed=0, rng=0, device=0, stream=None)
    a.update(change)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(dtype=L.FO_F32), b"fp16 or bf16"), (dict(table=None), b"null"), (dict(table_dtype=L.FO_F16), b"table"),
    (dict(table=18), b"aligned"), (dict(ts=(ctypes.c_int64 * 2)(-1, 1)), b"strides"),
    (dict(starts=starts_array(1, 2)[0], n=2), b"distance 0"), (dict(starts=starts_array(0, 3, 2)[0], n=3), b"descend"),
    (dict(n=0), b"buckets"), (dict(n=257), b"buckets"), (dict(offset=-1), b"query_offset"), (dict(offset=2**29 + 1), b"query_offset"),
    (dict(Sq=0), b"Sq"), (dict(workspace=None), b"workspace"), (dict(workspace=24), b"workspace"), (dict(B=0), b"positive"),
    (dict(p=1.0), b"dropout_p"), (dict(bias=16), b"strides"), (dict(scale=0.0), b"scale"), (dict(scale=1e-30), b"scale"),
    (dict(bias=16, bs=(ctypes.c_int64 * 3)(0, 0, 8)), b"row stride"),
    (dict(bias=16, bs=(ctypes.c_int64 * 3)(0, 0, 0), bias_dtype=L.FO_F16), b"bias"), (dict(D=60), b"head_dim"),
])
def test_the_forward_entry_validates_before_any_cuda_call(change, message):
    lib = L.load()
    assert lib.fo_rel_attn_fwd(*forward_args(lib, **change).values()) == -1
    assert message in lib.fo_last_error(), lib.fo_last_error()


def test_the_backward_entry_validates_before_any_cuda_call():
    lib = L.load()
    s = (ctypes.c_int64 * 3)(8 * 64 * 2, 8 * 64, 64)
    starts, n = starts_array(0, 1, 2, 5)

    def call(dtable=16, partials=16, workspace=16, scale=0.125, table_dtype=L.FO_F32, delta=16):
        return lib.fo_rel_attn_bwd(16, 16, 16, 16, 16, 16, 16, 16, 16, dtable, 16, delta, partials, 1, 2, 8, 8, 64, *([s] * 8),
                                   L.FO_BF16, 0, scale, table_dtype, starts, n, 1, 0, workspace, None, None, L.FO_F32, 0.0, 0, 0, 0,
                                   None)

    for change, message in ((dict(partials=None), b"workspace"), (dict(partials=20), b"partials"), (dict(workspace=None), b"null"),
                            (dict(workspace=20), b"workspace"), (dict(table_dtype=L.FO_F16), b"table"), (dict(dtable=18), b"dtable"),
                            (dict(scale=-1.0), b"scale"), (dict(delta=None), b"null")):
        assert call(**change) == -1
        assert message in lib.fo_last_error(), (change, lib.fo_last_error())


def test_workspace_sizes():
    lib = L.load()
    starts, n = starts_array(*relative_bucket_starts(32, 128, True))
    one = lib.fo_rel_attn_workspace(1, 1000, 1000, starts, n, 1, 0, 0)
    assert 0 < one < 64 * 1024
    assert lib.fo_rel_attn_workspace(12, 1000, 1000, starts, n, 1, 0, 0) > one
    assert lib.fo_rel_attn_workspace(1, 1000, 1000, starts, n, 1, 0, 7) >= one + 7 * 4000
    assert lib.fo_rel_attn_workspace(0, 1000, 1000, starts, n, 1, 0, 0) == -1
    assert lib.fo_rel_attn_workspace(1, 1000, 1000, starts, n, 1, 0, -1) == -1
    assert lib.fo_rel_attn_bwd_workspace(2, 3, 256, 384, 64, 32, 0) > 0
    assert lib.fo_rel_attn_bwd_workspace(2, 3, 0, 384, 64, 32, 0) == -1


def test_norm_entry_validates_before_any_cuda_call():
    lib = L.load()
    ptr, num, dt = (ctypes.c_void_p * 1)(16), (ctypes.c_int64 * 1)(8), (ctypes.c_int * 1)(L.FO_F32)
    assert lib.fo_grad_norm(ptr, num, dt, -1, 1.0, 16, None, 16, None, 0, None) == -1
    assert lib.fo_grad_norm(ptr, num, dt, 1, -1.0, 16, None, 16, None, 0, None) == -1 and b"max_norm" in lib.fo_last_error()
    assert lib.fo_grad_norm(ptr, num, (ctypes.c_int * 1)(5), 1, 1.0, 16, None, 16, None, 0, None) == -1 and b"dtype" in lib.fo_last_error()
    assert lib.fo_grad_norm(ptr, (ctypes.c_int64 * 1)(1 << 45), dt, 1, 1.0, 16, None, 16, None, 0, None) == -1
    assert lib.fo_grad_norm(ptr, num, dt, 1, 1.0, 16, None, None, None, 0, None) == -1
    assert lib.fo_grad_norm_workspace(1) > 0 and lib.fo_grad_norm_workspace(3000) > lib.fo_grad_norm_workspace(1000)
    s = (ctypes.c_void_p * 1)(16)
    args = (s, s, s, num, 1, L.FO_F32, L.FO_F32, L.FO_F32, 1e-3, 0.9, 0.99, 0.0)
    assert lib.fo_lion_multi_tensor_step_clipped(*args, None, 0, None) == -1 and b"clipping" in lib.fo_last_error()
    assert lib.fo_lion_flat_step_clipped(16, 16, 16, 0, 8, L.FO_F32, L.FO_F32, L.FO_F32, 1e-3, 0.9, 0.99, 0.0, None, 0, None) == -1
