"""How far the gradient of a relative bias table may be off: a statistical bound, and the cases it is used at.

The kernels sum dS unrounded, so what the table's gradient is off by comes from delta = rowsum(O o dO): O is rounded
to the input type, and so is the P it was summed from.  Every rounding is off by at most e = finfo(dtype).eps / 2 of its
value, is as often up as down and does not depend on the others, so the error of a row's delta has the variance

    sigma_i^2 = sum_d (e O_id dO_id)^2 / 3 + sum_j (e P_ij dP_ij)^2 / 3      (uniform within a half step)

It leaves P_ij times that error, with one sign, in every dS of the row.  A bucket u gets the error times P_iu, the row's
probability in u, less what the correction of the far sums takes out: a share of the row's error that is at most
the largest far probability of a row in the same block of queries.  Both lie within the largest P_iu of the rows of the
128-row tile, q_iu, and their difference within it too, so that, with the tiles' far sums of all rows independent,

    |error of dT_u| <= 6 sqrt(sum_i sigma_i^2 q_iu^2) + F sum_ij in u P_ij (|dP_ij| + |delta_i|) + half a step of dT_u

6 deviations, and F = 2^-16 for the fp32 arithmetic as in the elementwise bounds.  The 2-norm over the buckets of each
head is compared with the 2-norm of these.  Far sums left out, taken twice or with the wrong sign are several times that:
test_table_gradient_bound_cpu.py shows so for each case.
"""
import math

import torch

F32 = 2.0**-16


def bucket_ids(M, N, num_buckets, max_distance, bidirectional, offset):
    half = num_buckets // 2 if bidirectional else num_buckets
    near = half // 2
    d = torch.arange(N)[None, :] - torch.arange(M)[:, None] - offset
    n = d.abs() if bidirectional else (-d).clamp(min=0)
    far = torch.log(n.clamp(min=1).double() / near) / math.log(max_distance / near) * (half - near)
    ids = torch.where(n < near, n, (near + torch.floor(far + 1e-9).long()).clamp(max=half - 1))
    return ids + (half * (d > 0) if bidirectional else 0)


def far_parts(M, N, num_buckets, max_distance, bidirectional, offset, cols):
    """Which pairs lie in a part of 32 keys x `cols` queries that is wholly beyond the last bucket's start: those whose
    gradient comes from the sums over parts."""
    half = num_buckets // 2 if bidirectional else num_buckets
    near = half // 2
    last = near
    steps = half - near
    while last**steps < max_distance ** (steps - 1) * near:  # the start of the last bucket
        last += 1
    first_key = torch.arange(N) // 32 * 32
    first_query = torch.arange(M) // cols * cols + offset
    lo = first_key[None, :] - (first_query + cols - 1)[:, None]
    hi = first_key[None, :] + 31 - first_query[:, None]
    left = hi <= -min(last, M + offset)
    right = lo >= (min(max(last, 1), N) if bidirectional else 0)
    return left | right


def expected(Q, K, V, table, dO, *, max_distance, bidirectional, offset=0, causal=False, bias=None, keep=None, p_drop=0.0,
             drop_pairs=None):
    """(dT, bound), both (num_buckets, H) in 64 bits.  `drop_pairs`: pairs whose part is left out of dT."""
    B, H, M, D = Q.shape
    N, dev = K.shape[2], Q.device
    e = torch.finfo(Q.dtype).eps / 2
    q, k, v, g = Q.double(), K.double(), V.double(), dO.double()
    ids = bucket_ids(M, N, table.shape[0], max_distance, bidirectional, offset).to(dev)
    s = q @ k.transpose(2, 3) / math.sqrt(D) + table.double()[ids].permute(2, 0, 1)
    if bias is not None:
        b64 = bias.double()
        s = s + torch.where(b64 <= -1e6, torch.full_like(b64, -math.inf), b64)
    if causal:
        s = s.masked_fill(torch.arange(N, device=dev)[None, :] > torch.arange(M, device=dev)[:, None] + offset, -math.inf)
    p = torch.softmax(s, dim=-1).nan_to_num(0.0)
    m = 1.0 if keep is None else keep.double() / (1 - p_drop)
    dp = (g @ v.transpose(2, 3)) * m
    O = (p * m) @ v
    delta = (g * O).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    variance = ((e * O * g).square().sum(-1) + (e * p * dp).square().sum(-1)) / 3
    flat = ids.reshape(-1)
    u = table.shape[0]

    def by_bucket(x):  # (..., M, N) summed by bucket: (u, ...)
        return torch.zeros(u, x[..., 0, 0].numel(), dtype=torch.float64, device=dev).index_add_(
            0, flat, x.reshape(-1, M * N).T.contiguous()).view(u, *x.shape[:-2])

    rows = torch.zeros(B, H, M, u, dtype=torch.float64, device=dev).scatter_add_(3, ids.expand(B, H, M, N).contiguous(), p)
    tiles = torch.nn.functional.pad(rows, (0, 0, 0, -M % 128)).view(B, H, -1, 128, u)
    largest = tiles.amax(3, keepdim=True).expand_as(tiles).reshape(B, H, -1, u)[:, :, :M]
    spread = (variance[..., None] * largest.square()).sum((0, 2)).sqrt().T
    arithmetic = F32 * by_bucket((p * (dp.abs() + delta.abs())).sum(0))
    if drop_pairs is not None:
        ds = ds.masked_fill(drop_pairs.to(dev), 0.0)
    dT = by_bucket(ds.sum(0))
    return dT, 6 * spread + arithmetic + torch.finfo(table.dtype).eps / 2 * dT.abs()


#: (name, B, H, M, N, D, dtype, num_buckets, max_distance, bidirectional, offset, lens of the keys or "holes", dropout)
BF, HF = torch.bfloat16, torch.float16
CASES = [
    ("batches", 3, 4, 700, 700, 64, BF, 32, 128, True, 0, None, 0.0),
    ("batches one-sided", 4, 4, 900, 900, 64, BF, 16, 40, False, 0, None, 0.0),
    ("two-sided width 96", 2, 4, 700, 700, 96, BF, 16, 40, True, 0, None, 0.0),
    ("one-sided width 80, fp16", 2, 4, 701, 701, 80, HF, 16, 40, False, 0, None, 0.0),
    ("D 128 fp16", 2, 4, 650, 900, 128, HF, 16, 40, True, 0, None, 0.0),
    ("more keys than queries", 2, 4, 333, 1100, 64, BF, 16, 40, True, 0, None, 0.0),
    ("more queries than keys", 2, 4, 1100, 333, 128, BF, 16, 40, True, 0, None, 0.0),
    ("the last queries", 3, 4, 200, 1000, 64, BF, 32, 128, False, 800, None, 0.0),
    ("a chunk, two-sided", 3, 4, 257, 1000, 128, BF, 16, 40, True, 371, None, 0.0),
    ("padding", 3, 4, 600, 800, 64, BF, 16, 40, True, 0, (800, 511, 640), 0.0),
    ("padding, one-sided D 128", 3, 4, 800, 800, 128, BF, 16, 40, False, 0, (800, 300, 777), 0.0),
    ("holes", 3, 4, 600, 900, 64, HF, 16, 40, True, 0, "holes", 0.0),
    ("holes, offset, D 96", 3, 4, 330, 900, 96, BF, 16, 40, False, 570, "holes", 0.0),
    ("dropout", 2, 4, 700, 700, 64, BF, 16, 40, True, 0, None, 0.2),
    ("dropout D 128", 3, 4, 700, 700, 128, BF, 16, 40, True, 0, None, 0.1),
    ("dropout D 128, padding, offset", 3, 4, 400, 900, 128, BF, 16, 40, False, 500, (900, 700, 850), 0.1),
    ("dropout, holes, fp16", 3, 4, 640, 900, 64, HF, 16, 40, True, 0, "holes", 0.3),
]


def inputs(case, device):
    """(Q, K, V, table, dO, keywords of the call without dropout's, dropout)."""
    _, B, H, M, N, D, dtype, nb, md, bid, offset, lens, p = case
    gen = torch.Generator().manual_seed(M + N + D)
    r = lambda *s: torch.empty(s).normal_(generator=gen).to(dtype).to(device)  # noqa: E731
    table = torch.empty(nb, H).normal_(generator=gen).to(device)
    bias = None
    if lens is not None:
        bias = torch.zeros(B, 1, 1, N)
        if lens == "holes":
            bias[0, ..., N // 2:] = -math.inf
            bias[1, ..., :200] = -math.inf
            bias[1, ..., 333:520] = -math.inf
            bias[2] = torch.linspace(-1, 1, N)
        else:
            for b in range(B):
                bias[b, ..., lens[b]:] = -math.inf
        bias = bias.to(device)
    kw = dict(max_distance=md, bidirectional=bid, causal=not bid, bias=bias)
    return r(B, H, M, D), r(B, H, N, D), r(B, H, N, D), table, r(B, H, M, D), kw, offset, p
