"""Attention with a learned relative position bias against the formula in 64 bits.

Tolerances.  The kernels round P and dS to the 16-bit input type before their matmuls (half a step each:
e = finfo(dtype).eps / 2 relative), every result once more, and keep everything else in fp32; F = 2^-16
relative covers fp32 (exp2 to 2^-22, LSE of a few units to 2^-21, sums of at most a few thousand products).
So, elementwise, with |.| of the 64-bit quantities:
  O       (e |O|) + (e + F) P |V|
  dV      e |dV| + (e + F) P^T |dO|
  dS      E = e |dS| + F P (|dP| + |delta|) + P w,  where w bounds the error of delta = rowsum(O o dO), O's
          own rounding and that of the P it was summed from: e |O| |dO| + (e + F) P |V| |dO|
  dQ, dK  e |.| + scale (E |K|), scale (E^T |Q|)
  dTable  half a step of its type + the sum of E - e |dS| over the bucket (dS is summed unrounded).  What w
          stands for is mostly taken out again (the sums over a block of queries are made to be zero), which
          moves another side's share to a bucket: at most as much again
fp16 products that fall below 6e-5 lose half of 2^-24 absolutely: added where P is rounded.
"""
import math

import pytest
import torch

import fast_ops_b200._lib as L
from fast_ops_b200.flash_attention import (
    dropout_mask,
    multi_head_attention,
    relative_attention,
    relative_bucket_starts,
)

pytestmark = pytest.mark.gpu
F32 = 2.0**-16


def bucket_ids(M, N, num_buckets, max_distance, bidirectional, offset, device):
    """The definition, from real numbers: floor of the logarithm's share, borders by exact integers."""
    half = num_buckets // 2 if bidirectional else num_buckets
    near = half // 2
    d = torch.arange(N)[None, :] - torch.arange(M)[:, None] - offset
    n = d.abs() if bidirectional else (-d).clamp(min=0)
    far = torch.log(n.clamp(min=1).double() / near) / math.log(max_distance / near) * (half - near)
    ids = torch.where(n < near, n, (near + torch.floor(far + 1e-9).long()).clamp(max=half - 1))
    return (ids + (half * (d > 0) if bidirectional else 0)).to(device)


def formula(Q, K, V, table, dO, *, max_distance, bidirectional, offset=0, causal=False, bias=None, keep=None, p_drop=0.0,
            scale=None):
    """Results and error bounds in 64 bits; rows without keys give zeros."""
    B, H, M, D = Q.shape
    N = K.shape[2]
    dt, dev = Q.dtype, Q.device
    e = torch.finfo(dt).eps / 2
    tiny = 2.0**-25 if dt == torch.float16 else 0.0
    q, k, v, t = Q.double(), K.double(), V.double(), table.double()
    scale = 1 / math.sqrt(D) if scale is None else scale
    ids = bucket_ids(M, N, table.shape[0], max_distance, bidirectional, offset, dev)
    s = q @ k.transpose(2, 3) * scale + t[ids].permute(2, 0, 1)
    if bias is not None:
        b64 = bias.double()
        s = s + torch.where(b64 <= -1e6, torch.full_like(b64, -math.inf), b64)
    if causal:
        hidden = torch.arange(N, device=dev)[None, :] > torch.arange(M, device=dev)[:, None] + offset
        s = s.masked_fill(hidden, -math.inf)
    p = torch.softmax(s, dim=-1).nan_to_num(0.0)
    lse = torch.logsumexp(s, dim=-1)
    m = 1.0 if keep is None else keep.double() / (1 - p_drop)
    pd = p * m
    out = {"O": pd @ v, "LSE": lse, "P": p}
    tol = {"O": e * out["O"].abs() + (e + F32) * (pd @ v.abs()) + tiny * N * v.abs().amax()}
    if dO is None:
        return out, tol
    g = dO.double()
    dp = (g @ v.transpose(2, 3)) * m
    delta = (g * out["O"]).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    size = (g.abs() * out["O"].abs()).sum(-1, keepdim=True)
    w = e * size + (e + F32) * (pd * (g.abs() @ v.abs().transpose(2, 3))).sum(-1, keepdim=True)
    E0 = F32 * p * ((g.abs() @ v.abs().transpose(2, 3)) * m + delta.abs()) + p * w
    E = e * ds.abs() + E0 + tiny
    out |= {"dV": pd.transpose(2, 3) @ g, "dQ": ds @ k * scale, "dK": ds.transpose(2, 3) @ q * scale}
    tol["dV"] = e * out["dV"].abs() + (e + F32) * (pd.transpose(2, 3) @ g.abs()) + tiny * M * g.abs().amax()
    tol["dQ"] = e * out["dQ"].abs() + scale * (E @ k.abs())
    tol["dK"] = e * out["dK"].abs() + scale * (E.transpose(2, 3) @ q.abs())
    dt_sum, e_sum = ds.sum(0), 2 * E0.sum(0)
    flat = ids.reshape(-1)
    out["dT"], tol["dT"] = (torch.zeros(table.shape[0], H, dtype=torch.float64, device=dev).index_add_(
        0, flat, x.reshape(H, -1).T.contiguous()) for x in (dt_sum, e_sum))
    tol["dT"] = tol["dT"] + torch.finfo(table.dtype).eps / 2 * out["dT"].abs() + 1e-30
    return out, tol


def close(name, got, want, tol):
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), f"{name}: not finite"
    off = (got.double() - want).abs() / tol.clamp(min=1e-37)
    assert off.max().item() <= 1.0, f"{name}: {off.max().item():.3f} of the tolerance at {off.argmax().item()}"


def make(B, H, M, N, D, dtype, num_buckets, table_dtype=None, seed=0, device="cuda", kv_heads=None):
    gen = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.empty(s, dtype=dtype, device=device).normal_(generator=gen)  # noqa: E731
    table = torch.empty(num_buckets, H, device=device).normal_(generator=gen).to(table_dtype or dtype)
    kv = kv_heads or H
    return r(B, H, M, D), r(B, kv, N, D), r(B, kv, N, D), table, r(B, H, M, D)


def padding(B, N, lens, device="cuda", value=-math.inf, dtype=torch.float32):
    keys = torch.arange(N, device=device)
    lens = torch.tensor([lens[i % len(lens)] for i in range(B)], device=device)
    return torch.zeros(B, N, device=device, dtype=dtype).masked_fill(keys >= lens[:, None], value).view(B, 1, 1, N)


def train(Q, K, V, table, dO, **kw):
    leaves = [t.detach().clone().requires_grad_() for t in (Q, K, V, table)]
    O, lse = relative_attention(*leaves, return_lse=True, **kw)
    return (O, lse) + torch.autograd.grad(O, leaves, dO)


def check_train(Q, K, V, table, dO, keep=None, **kw):
    got = train(Q, K, V, table, dO, **kw)
    t = table.detach().clone().requires_grad_()
    want, tol = formula(Q, K, V, t, dO, max_distance=kw["max_distance"], bidirectional=kw["bidirectional"],
                        offset=kw.get("query_offset", 0), causal=kw.get("causal", False), bias=kw.get("bias"), keep=keep,
                        p_drop=kw.get("dropout_p", 0.0), scale=kw.get("softmax_scale"))
    want, tol = ({n: x.detach() for n, x in d.items()} for d in (want, tol))
    close("O", got[0].detach(), want["O"], tol["O"])
    seen = want["LSE"] > -math.inf
    assert torch.equal(got[1] > -math.inf, seen)
    assert (got[1].double() - want["LSE"])[seen].abs().max().item() <= 2e-5 if seen.any() else True
    for name, x in zip(("dQ", "dK", "dV", "dT"), got[2:]):
        close(name, x, want[name], tol[name])
    torch.cuda.synchronize()
    assert L.device_status(0) == 0
    return got


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("B,H,M,N,D,dtype,nb,md,bid,causal,offset", [
    (1, 1, 1, 1, 64, BF, 32, 128, True, False, 0),
    (1, 2, 2, 3, 64, BF, 4, 2, True, False, 0),
    (2, 3, 64, 64, 64, BF, 32, 128, True, False, 0),
    (2, 3, 65, 127, 64, HF, 32, 128, True, False, 0),
    (1, 2, 128, 129, 128, BF, 32, 128, False, True, 0),
    (1, 2, 257, 257, 128, HF, 16, 40, False, True, 0),
    (2, 2, 300, 513, 80, BF, 64, 640, True, False, 0),
    (1, 2, 700, 700, 64, BF, 32, 128, True, False, 0),
    (1, 2, 700, 700, 64, BF, 32, 128, False, True, 0),
    (1, 2, 130, 700, 64, BF, 32, 128, False, True, 570),   # the last 130 of 700 positions
    (1, 2, 100, 700, 128, HF, 32, 128, False, True, 333),  # a chunk from the middle
    (1, 2, 33, 90, 40, BF, 32, 128, True, False, 5000),    # all keys far before the queries
    (1, 1, 900, 70, 8, BF, 32, 128, False, True, 0),       # more queries than keys
    (1, 1, 70, 900, 96, BF, 32, 128, False, True, 0),      # keys that no query sees
    (1, 2, 400, 400, 64, BF, 512, 4000, True, False, 0),   # every bucket near the diagonal
    (1, 1, 600, 600, 128, BF, 2, 600, False, True, 0),     # two buckets
    (1, 2, 640, 640, 64, HF, 32, 100000, True, False, 0),  # no constant far part
    (1, 2, 257, 300, 64, BF, 6, 3, True, False, 0),        # constant almost everywhere
])
@pytest.mark.parametrize("table_dtype", ["same", "fp32"])
def test_training_step_matches_the_formula(B, H, M, N, D, dtype, nb, md, bid, causal, offset, table_dtype, cuda_device):
    Q, K, V, table, dO = make(B, H, M, N, D, dtype, nb, FP if table_dtype == "fp32" else None, seed=M + N)
    check_train(Q, K, V, table, dO, max_distance=md, bidirectional=bid, causal=causal, query_offset=offset)


@pytest.mark.parametrize("lens", [(5,), (64, 0), (200, 129, 300)])
@pytest.mark.parametrize("D,dtype,bid,value,bias_dtype", [
    (64, BF, True, -math.inf, FP), (128, HF, True, -math.inf, HF), (64, BF, False, torch.finfo(FP).min, FP),
    (64, BF, True, torch.finfo(BF).min, BF), (128, BF, False, -1e9, FP)])
def test_padding_and_rows_without_keys(lens, D, dtype, bid, value, bias_dtype, cuda_device):
    B, H, M, N = 3, 2, 140, 300
    Q, K, V, table, dO = make(B, H, M, N, D, dtype, 32, seed=D)
    bias = padding(B, N, lens, value=value, dtype=bias_dtype)
    got = check_train(Q, K, V, table, dO, max_distance=128, bidirectional=bid, causal=not bid, bias=bias)
    for i in range(B):
        if lens[i % len(lens)] == 0:
            assert all((x[i] == 0).all() for x in (got[0], got[2], got[3], got[4]))


def test_a_head_wise_bias_and_a_broadcast_one(cuda_device):
    B, H, M, N, D = 2, 3, 200, 260, 64
    Q, K, V, table, dO = make(B, H, M, N, D, BF, 32, seed=5)
    for shape in ((1, H, 1, N), (B, H, 1, N), (1, 1, 1, N)):
        bias = torch.randn(shape, device="cuda")
        check_train(Q, K, V, table, dO, max_distance=128, bidirectional=True, bias=bias)
        strided = torch.randn(*shape[:3], 2 * N, device="cuda")[..., ::2]
        check_train(Q, K, V, table, dO, max_distance=128, bidirectional=True, bias=strided)
    check_train(Q, K, V, table, dO, max_distance=128, bidirectional=True, bias=torch.randn(1, 1, 1, N, device="cuda").expand(B, H, 1, N))


@pytest.mark.parametrize("D,dtype,padded,causal", [(64, BF, False, False), (128, HF, True, False), (64, HF, True, True), (128, BF, False, True)])
def test_dropout(D, dtype, padded, causal, cuda_device):
    B, H, M, N, p = 2, 2, 300, 300, 0.2
    Q, K, V, table, dO = make(B, H, M, N, D, dtype, 32, seed=9)
    rng = (1234, 48)
    keep = dropout_mask(p, B, H, M, N, Q.device, rng=rng)
    check_train(Q, K, V, table, dO, keep=keep, max_distance=128, bidirectional=not causal, causal=causal, dropout_p=p,
                rng=rng, bias=padding(B, N, (211, 300)) if padded else None)


def test_dropout_is_drawn_from_the_default_generator(cuda_device):
    Q, K, V, table, dO = make(2, 2, 96, 96, 64, BF, 32)
    torch.cuda.manual_seed(7)
    keep = dropout_mask(0.3, 2, 2, 96, 96, Q.device)
    after = torch.cuda.get_rng_state()
    torch.cuda.manual_seed(7)
    check_train(Q, K, V, table, dO, keep=keep, max_distance=128, bidirectional=True, dropout_p=0.3)
    assert torch.equal(torch.cuda.get_rng_state(), after)


@pytest.mark.parametrize("B,H,N,D,dtype,nb,md,bid,offset,kv", [
    (1, 1, 1, 64, BF, 32, 128, False, 0, 1),
    (3, 5, 77, 64, HF, 32, 128, False, 76, 5),
    (2, 4, 1000, 128, BF, 32, 128, False, 999, 4),
    (2, 6, 513, 128, BF, 16, 50, False, 512, 1),     # one K/V head for all
    (5, 7, 300, 64, BF, 32, 128, True, 100, 1),      # keys behind the query too
    (2, 3, 4097, 80, HF, 64, 2000, False, 4096, 3),
    (1, 2, 3000, 8, BF, 32, 128, False, 123456, 2),  # a window of keys long before the query
    (1, 2, 500, 128, BF, 512, 1000, True, 250, 2),
])
@pytest.mark.parametrize("padded", [False, True])
def test_single_token(B, H, N, D, dtype, nb, md, bid, offset, kv, padded, cuda_device):
    Q, K, V, table, _ = make(B, H, 1, N, D, dtype, nb, seed=N, kv_heads=kv)
    K, V = (t.expand(B, H, N, D) for t in (K, V))
    bias = padding(B, N, (N, max(1, N // 3), 0)) if padded else None
    O, lse = relative_attention(Q, K, V, table, max_distance=md, bidirectional=bid, query_offset=offset, bias=bias,
                                return_lse=True)
    want, tol = formula(Q, K, V, table, None, max_distance=md, bidirectional=bid, offset=offset, bias=bias)
    close("O", O, want["O"], tol["O"])
    seen = want["LSE"] > -math.inf
    assert torch.equal(lse > -math.inf, seen)
    assert not seen.any() or (lse.double() - want["LSE"])[seen].abs().max().item() <= 2e-5
    assert (O[~seen] == 0).all()


def test_single_token_with_a_causal_mask_sees_keys_up_to_its_position(cuda_device):
    Q, K, V, table, _ = make(2, 3, 1, 400, 64, BF, 32)
    for offset in (0, 1, 250, 399, 1000):
        O = relative_attention(Q, K, V, table, bidirectional=False, query_offset=offset, causal=True)
        want, tol = formula(Q, K, V, table, None, max_distance=128, bidirectional=False, offset=offset, causal=True)
        close("O", O, want["O"], tol["O"])


def test_decoding_token_by_token_agrees_with_the_whole_sequence(cuda_device):
    B, H, N, D = 2, 4, 150, 64
    Q, K, V, table, _ = make(B, H, N, N, D, BF, 32)
    want, tol = formula(Q, K, V, table, None, max_distance=128, bidirectional=False, causal=True)
    whole = relative_attention(Q, K, V, table, bidirectional=False, causal=True)
    close("O", whole, want["O"], tol["O"])
    for i in (0, 1, 77, 149):
        one = relative_attention(Q[:, :, i:i + 1], K[:, :, :i + 1], V[:, :, :i + 1], table, bidirectional=False, query_offset=i)
        close(f"row {i}", one, want["O"][:, :, i:i + 1], tol["O"][:, :, i:i + 1])


def test_shared_key_value_heads_and_transposed_layouts(cuda_device):
    B, H, M, N, D = 2, 4, 150, 200, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.empty(s, dtype=BF, device="cuda").normal_(generator=gen)  # noqa: E731
    q, k1, v1 = r(B, M, H, D), r(B, N, 1, D), r(B, N, 1, D)
    table, dO = r(32, H), r(B, M, H, D)
    leaves = [t.clone().requires_grad_() for t in (q, k1, v1, table)]
    O = relative_attention(leaves[0].transpose(1, 2), leaves[1].transpose(1, 2).expand(B, H, N, D),
                           leaves[2].transpose(1, 2).expand(B, H, N, D), leaves[3])
    dq, dk, dv, dt = torch.autograd.grad(O, leaves, dO.transpose(1, 2))
    Q, K, V = q.transpose(1, 2), k1.transpose(1, 2).expand(B, H, N, D), v1.transpose(1, 2).expand(B, H, N, D)
    want, tol = formula(Q, K, V, table.clone().requires_grad_(), dO.transpose(1, 2), max_distance=128, bidirectional=True)
    want, tol = ({n: x.detach() for n, x in d.items()} for d in (want, tol))
    e = torch.finfo(BF).eps / 2
    close("O", O.detach(), want["O"], tol["O"])
    close("dQ", dq.transpose(1, 2), want["dQ"], tol["dQ"])
    close("dT", dt, want["dT"], tol["dT"])
    for name, got in (("dK", dk), ("dV", dv)):
        # autograd sums the heads' rounded gradients and rounds the sum
        total = want[name].sum(1, keepdim=True)
        bound = tol[name].sum(1, keepdim=True) + H * e * want[name].abs().sum(1, keepdim=True)
        close(name, got.transpose(1, 2), total, bound)


def test_a_table_with_strides_and_one_shared_by_the_heads(cuda_device):
    B, H, M, N, D = 1, 3, 140, 180, 64
    Q, K, V, _, dO = make(B, H, M, N, D, BF, 32)
    wide = torch.randn(H, 64, device="cuda")
    table = wide.T[::2]  # strides (2, 64)
    check_train(Q, K, V, table.clone(), dO, max_distance=128, bidirectional=True)
    a = relative_attention(Q, K, V, table)
    assert torch.equal(a, relative_attention(Q, K, V, table.contiguous()))
    shared = torch.randn(32, 1, device="cuda", requires_grad=True)
    O = relative_attention(Q, K, V, shared.expand(32, H))
    g, = torch.autograd.grad(O, shared, dO)
    want, tol = formula(Q, K, V, shared.detach().expand(32, H).clone().requires_grad_(), dO, max_distance=128, bidirectional=True)
    close("dT", g, want["dT"].detach().sum(1, keepdim=True), tol["dT"].detach().sum(1, keepdim=True) * 1.01)


def test_only_the_gradients_that_are_asked_for(cuda_device):
    Q, K, V, table, dO = make(1, 2, 130, 130, 64, BF, 32)
    full = train(Q, K, V, table, dO)
    t = table.clone().requires_grad_()
    g, = torch.autograd.grad(relative_attention(Q, K, V, t), t, dO)
    assert torch.equal(g, full[5])  # the same bits from run to run
    q = Q.clone().requires_grad_()
    g, = torch.autograd.grad(relative_attention(q, K, V, table), q, dO)
    want, tol = formula(Q, K, V, table, dO, max_distance=128, bidirectional=True)
    close("dQ", g, want["dQ"], tol["dQ"])


def test_the_table_gradient_agrees_with_differences(cuda_device):
    """d/dt of sum(O o dO), by central differences of the formula in 64 bits, for a few entries."""
    Q, K, V, table, dO = make(1, 2, 90, 110, 64, HF, 32, FP, seed=1)
    dT = train(Q, K, V, table, dO)[5]
    _, tol = formula(Q, K, V, table.clone().requires_grad_(), dO, max_distance=128, bidirectional=True)
    h = 1e-4
    for u, head in ((0, 0), (3, 1), (12, 0), (17, 1), (25, 0)):
        at = []
        for sign in (1, -1):
            t = table.double().clone()
            t[u, head] += sign * h
            at.append((formula(Q, K, V, t, None, max_distance=128, bidirectional=True)[0]["O"] * dO.double()).sum().item())
        diff = (at[0] - at[1]) / (2 * h)
        # the third derivative of a softmax average is below 6 times its range
        slack = tol["dT"][u, head].item() + h * h * 6 * V.double().abs().max().item() * dO.double().abs().sum().item() / 6
        assert abs(dT[u, head].item() - diff) <= slack


@pytest.mark.parametrize("N,D,dtype,nb,md,bid", [(2048, 64, BF, 16, 32, True), (2048, 128, BF, 32, 128, False), (1500, 64, HF, 32, 128, True)])
def test_far_buckets_keep_their_precision(N, D, dtype, nb, md, bid, cuda_device):
    """The far buckets sum thousands of terms that nearly cancel; an error of delta, the same for all keys of
    a query, does not.  All in all the table's gradient is to lose no more than a rounding of it to the
    input type would: e of its 2-norm (without the correction of the sums it is 2 to 3 e here)."""
    Q, K, V, table, dO = make(1, 4, N, N, D, dtype, nb, FP, seed=N)
    dT = train(Q, K, V, table, dO, max_distance=md, bidirectional=bid, causal=not bid)[5]
    want, _ = formula(Q, K, V, table, dO, max_distance=md, bidirectional=bid, causal=not bid)
    off = (dT.double() - want["dT"]).norm() / want["dT"].norm()
    assert off.item() <= torch.finfo(dtype).eps / 2


def test_a_table_of_zeros_is_plain_attention(cuda_device):
    Q, K, V, table, dO = make(2, 2, 333, 333, 64, BF, 32)
    zero = torch.zeros_like(table)
    got = train(Q, K, V, zero, dO)
    leaves = [t.clone().requires_grad_() for t in (Q, K, V)]
    O = multi_head_attention(*leaves, causal=False)
    want, tol = formula(Q, K, V, zero.clone().requires_grad_(), dO, max_distance=128, bidirectional=True)
    for a, b, n in zip(got[:1] + got[2:5], (O,) + torch.autograd.grad(O, leaves, dO), ("O", "dQ", "dK", "dV")):
        e = torch.finfo(BF).eps / 2
        bound = 2 * tol[n].detach() + (0 if n in ("O", "dV") else 2 * e) * want[n].detach().abs().amax()
        assert ((a.detach().double() - b.detach().double()).abs() <= bound).all(), n


def test_masked_buckets(cuda_device):
    """A table entry of -inf hides its keys: here all but a window of 8 keys up to the query's own."""
    Q, K, V, table, dO = make(1, 2, 200, 200, 64, BF, 32)
    table[8:] = -math.inf
    got = train(Q, K, V, table, dO, max_distance=128, bidirectional=False, causal=True)
    t = table.clone().requires_grad_()
    want, tol = formula(Q, K, V, t, dO, max_distance=128, bidirectional=False, causal=True)
    for name, x in zip(("O", "dQ", "dK", "dV", "dT"), got[:1] + got[2:]):
        close(name, x.detach(), want[name].detach(), tol[name].detach())
    assert (got[5][8:] == 0).all()


def test_other_streams_and_graph_replay(cuda_device):
    Q, K, V, table, dO = make(2, 2, 256, 256, 64, BF, 32)
    want = train(Q, K, V, table, dO)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train(Q, K, V, table, dO)
    side.synchronize()
    for i in (0, 1, 5):
        assert torch.equal(got[i], want[i])
    # forward and decoding form in a graph, replayed on new inputs
    q, k, v, t = (x.clone() for x in (Q, K, V, table))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.no_grad(), torch.cuda.graph(graph):
        o = relative_attention(q, k, v, t)
        o1 = relative_attention(q[:, :, :1], k, v, t, bidirectional=False, query_offset=255)
    Q2, K2, V2, t2, _ = make(2, 2, 256, 256, 64, BF, 32, seed=8)
    for dst, src in ((q, Q2), (k, K2), (v, V2), (t, t2)):
        dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, relative_attention(Q2, K2, V2, t2))
    assert torch.equal(o1, relative_attention(Q2[:, :, :1], K2, V2, t2, bidirectional=False, query_offset=255))


def test_a_training_step_in_a_graph(cuda_device):
    Q, K, V, table, dO = make(2, 2, 200, 200, 64, BF, 32)
    leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(relative_attention(*leaves), leaves, dO)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        O = relative_attention(*leaves)
        grads = torch.autograd.grad(O, leaves, dO)
    other = make(2, 2, 200, 200, 64, BF, 32, seed=4)
    with torch.no_grad():
        for dst, src in zip(leaves, other):
            dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    want, tol = formula(*other[:3], other[3].clone().requires_grad_(), dO, max_distance=128, bidirectional=True)
    for name, x in zip(("O", "dQ", "dK", "dV", "dT"), (O,) + grads):
        close(name, x.detach(), want[name].detach(), tol[name].detach())


def test_long_sequences_by_blocks(cuda_device):
    """Positions far apart: 9000 keys, checked on a few rows of one head."""
    B, H, N, D = 1, 2, 9000, 128
    Q, K, V, table, _ = make(B, H, N, N, D, BF, 32)
    O = relative_attention(Q, K, V, table, bidirectional=False, causal=True)
    for rows in (slice(0, 130), slice(4400, 4500), slice(8930, 9000)):
        q = Q[:, :, rows]
        want, tol = formula(q, K, V, table, None, max_distance=128, bidirectional=False, offset=rows.start, causal=True)
        close(f"rows {rows.start}", O[:, :, rows], want["O"], tol["O"])


def test_refusals(cuda_device):
    Q, K, V, table, _ = make(2, 2, 64, 64, 64, BF, 32)
    ok = dict(max_distance=128)
    for bad in (
        lambda: relative_attention(Q, K, V, table[:, :1], **ok),
        lambda: relative_attention(Q, K, V, table[:31], **ok),
        lambda: relative_attention(Q, K, V, table.half(), **ok),
        lambda: relative_attention(Q, K, V, table.cpu(), **ok),
        lambda: relative_attention(Q, K, V, table, max_distance=8),
        lambda: relative_attention(Q, K, V, table, query_offset=-1),
        lambda: relative_attention(Q, K, V, table, bias=torch.zeros(1, 1, 64, 64, device="cuda")),
        lambda: relative_attention(Q, K, V, table, bias=torch.zeros(1, 1, 1, 63, device="cuda")),
        lambda: relative_attention(Q, K, V, table, bias=torch.zeros(1, 1, 1, 64, device="cuda", requires_grad=True)),
        lambda: relative_attention(Q, K, V, table, dropout_p=1.0),
        lambda: relative_attention(Q, K, V, table, softmax_scale=0.0),
        lambda: relative_attention(Q.float(), K.float(), V.float(), table),
        lambda: relative_attention(Q, K[:, :1], V[:, :1], table),
        lambda: relative_attention(Q[..., :60], K[..., :60], V[..., :60], table),
        lambda: relative_attention(Q.transpose(2, 3), K, V, table),
        lambda: relative_attention(Q, K[:, :, :0], V[:, :, :0], table),
    ):
        with pytest.raises(RuntimeError):
            bad()
    assert relative_bucket_starts(32, 128, True)[-1] == 91


@pytest.mark.parametrize("D,causal", [(64, False), (128, False), (64, True), (128, True)])
@pytest.mark.parametrize("dropout_p", [0.0, 0.1])
def test_masks_with_holes_and_ragged_ends(D, causal, dropout_p, cuda_device):
    """Keys masked in front, in the middle and at the end, whole key tiles of them, and values that are not masks."""
    B, H, M, N = 4, 2, 330, 700
    Q, K, V, table, dO = make(B, H, M, N, D, BF, 32, seed=2)
    bias = torch.zeros(B, 1, 1, N, device="cuda")
    bias[0, ..., 300:] = -math.inf
    bias[1, ..., :200] = -math.inf
    bias[1, ..., 250:520] = -math.inf
    bias[2, ..., 0] = 1.5
    bias[2, ..., 699] = -2.0
    bias[3] = torch.linspace(-3, 3, N, device="cuda")
    keep = dropout_mask(dropout_p, B, H, M, N, Q.device, rng=(5, 0)) if dropout_p else None
    check_train(Q, K, V, table, dO, keep=keep, max_distance=128, bidirectional=not causal, causal=causal, bias=bias,
                dropout_p=dropout_p, rng=(5, 0), query_offset=370 if causal else 0)


@pytest.mark.parametrize("impl", ["ws64", "ws64s"])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF), (96, BF)])
@pytest.mark.parametrize("causal", [False, True])
def test_both_forward_kernels(impl, D, dtype, causal, cuda_device):
    Q, K, V, table, dO = make(2, 3, 420, 420, D, dtype, 32, seed=6)
    L.attn_configure(impl=impl)
    try:
        for bias in (None, padding(2, 420, (300, 64))):
            check_train(Q, K, V, table, dO, max_distance=128, bidirectional=not causal, causal=causal, bias=bias)
    finally:
        L.attn_configure(impl="auto")


def test_output_gradients_that_are_broadcast_or_cut(cuda_device):
    Q, K, V, table, dO = make(2, 2, 100, 100, 64, BF, 32)
    leaves = [t.clone().requires_grad_() for t in (Q, K, V, table)]
    O = relative_attention(*leaves)
    for g in (torch.ones((), device="cuda", dtype=BF).expand_as(O), dO[:1].expand_as(O), dO[:, :, :1].expand_as(O),
              torch.randn(2, 2, 100, 65, device="cuda", dtype=BF)[..., 1:]):
        got = torch.autograd.grad(O, leaves, g, retain_graph=True)
        want = torch.autograd.grad(O, leaves, g.contiguous(), retain_graph=True)
        for i in (1, 2, 3):
            assert torch.equal(got[i], want[i])
        assert torch.allclose(got[0].float(), want[0].float(), rtol=2.0**-7, atol=1e-6)  # dQ is summed by atomic adds


def test_packed_projections(cuda_device):
    """Q, K and V as views of one (B, S, 3, H, D) tensor, whose gradient collects theirs."""
    B, H, S, D = 2, 3, 130, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.empty(B, S, 3, H, D, dtype=BF, device="cuda").normal_(generator=gen).requires_grad_()
    table = torch.empty(32, H, dtype=BF, device="cuda").normal_(generator=gen).requires_grad_()
    dO = torch.empty(B, H, S, D, dtype=BF, device="cuda").normal_(generator=gen)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    O = relative_attention(q, k, v, table)
    g, dT = torch.autograd.grad(O, (qkv, table), dO)
    want, tol = formula(*(t.detach().contiguous() for t in (q, k, v)), table, dO, max_distance=128, bidirectional=True)
    want, tol = ({n: x.detach() for n, x in d.items()} for d in (want, tol))
    close("O", O.detach(), want["O"], tol["O"])
    for i, name in enumerate(("dQ", "dK", "dV")):
        close(name, g[:, :, i].transpose(1, 2), want[name], tol[name])
    close("dT", dT, want["dT"], tol["dT"])


def test_two_streams_at_once(cuda_device):
    """Calls of different problems that run side by side share nothing."""
    problems = [make(2, 4, 500, 500, 64, BF, 32, seed=i) for i in range(2)]
    want = [train(*p) for p in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(train(*problems[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for x in (0, 1, 3, 4, 5):
                assert torch.equal(g[x], want[i][x])


def test_a_step_of_attention_clipping_and_lion(cuda_device):
    """The operators together, as a training loop uses them: attention with a learned bias, its table's gradient
    among those whose norm clips the step.  Each part against its formula from what the part before it gave."""
    from fast_ops_b200.lion import Lion

    B, H, S, D = 2, 4, 200, 64
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(B, S, H * D, dtype=BF, device="cuda").normal_(generator=gen)
    weights = [torch.nn.Parameter(torch.empty(H * D, H * D, dtype=BF, device="cuda").normal_(0, (H * D) ** -0.5, generator=gen))
               for _ in range(3)]
    table = torch.nn.Parameter(torch.empty(32, H, dtype=BF, device="cuda").normal_(generator=gen))
    params = weights + [table]
    opt = Lion(params, lr=1e-3, weight_decay=0.1, max_grad_norm=0.5)
    for step in range(3):
        q, k, v = ((x @ w.T).view(B, S, H, D).transpose(1, 2) for w in weights)
        O = relative_attention(q, k, v, table, bias=padding(B, S, (150, 200)), causal=False)
        dO = torch.empty_like(O).normal_(generator=gen)
        before = [p.detach().clone() for p in params]
        momenta = [opt.state[p]["exp_avg"].clone() if step else torch.zeros_like(p) for p in params]
        opt.zero_grad(set_to_none=True)
        O.backward(dO)
        want, tol = formula(*(t.detach().contiguous() for t in (q, k, v)), table.detach(), dO, max_distance=128,
                            bidirectional=True, bias=padding(B, S, (150, 200)))
        close("O", O.detach(), want["O"], tol["O"])
        close("dT", table.grad, want["dT"], tol["dT"])
        opt.step()
        norm = math.sqrt(sum(p.grad.double().square().sum().item() for p in params))
        assert abs(opt.grad_norm.item() - norm) <= 4.5 * 2.0**-24 * norm and norm > 0.5
        coef = torch.full((), 0.5, device="cuda") / (opt.grad_norm + 1e-6)
        for p, p0, m0 in zip(params, before, momenta):
            rp, rm = torch.nn.Parameter(p0), m0
            rp.grad = (p.grad.float() * coef).to(BF)
            ref = Lion([rp], lr=1e-3, weight_decay=0.1)
            ref.state[rp]["exp_avg"] = rm
            ref.step()
            assert torch.equal(p, rp) and torch.equal(opt.state[p]["exp_avg"], rm)
