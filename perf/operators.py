"""The training and decoding operators that are timed: attention with a learned relative position bias,
the global gradient norm, and the Lion step with clipping by that norm.

Where `own` is false, `run` computes them from elementary torch operations (their plain form, in 32
bits; sums over whole parameter lists and the bias table in 64), otherwise through this package's entry
points.  A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is
one pass, `work` the bytes and operations a pass cannot do without, `exact` the results in 64 bits.

Kinds of case:
  fwd    attention forward without gradients; with sq = 1 the decoding of one token per sequence, whose
         position is that of the last stored key
  train  attention forward and backward, as inside a training step; the table's gradient among the results
  norm   the 2-norm over all gradients of a list
  lion   one Lion step whose gradients are clipped to a global norm
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
FWD_SCORES_MOST = 1 << 30    # scores b * h * sq * sk of a drawn forward case, at most the largest listed one's
TRAIN_SCORES_MOST = 1 << 29  # the same for forward + backward
NUMEL_MOST = 300_000_000
BETAS = (0.9, 0.99)


def _attn(kind, name=None, *, b, h, sq, sk, d, dtype="bf16", buckets=32, distance=128, bidirectional=True,
          causal=False, padded=False):
    case = {"kind": kind, "b": b, "h": h, "sq": sq, "sk": sk, "d": d, "dtype": dtype, "buckets": buckets,
            "distance": distance, "bidirectional": bidirectional, "causal": causal, "padded": padded}
    if name:
        case["name"] = name
    return case


def _list(kind, name=None, *, shapes, param, momentum="bf16", tensors=0, smallest=0, largest=0):
    case = {"kind": kind, "shapes": shapes, "param": param, "momentum": momentum, "tensors": tensors,
            "smallest": smallest, "largest": largest}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # The smallest configured attention (B=2, H=4, S=256, head_dim 64): the call itself counts.
        _attn("fwd", "rel_fwd_small_f16", b=2, h=4, sq=256, sk=256, d=64, dtype="f16"),
        # One encoder layer over a batch of documents, padded to the longest of them.
        _attn("fwd", "rel_fwd_encoder", b=8, h=12, sq=1024, sk=1024, d=64, padded=True),
        # One decoder layer over a long prompt: the largest forward here.
        _attn("fwd", "rel_fwd_s8192_causal", b=1, h=16, sq=8192, sk=8192, d=128, bidirectional=False, causal=True),
        # Decoding one token for each of sixteen sequences with two thousand tokens of context.
        _attn("fwd", "rel_decode_b16_k2048", b=16, h=12, sq=1, sk=2048, d=64, bidirectional=False),
        # Decoding against a long context, wide heads.
        _attn("fwd", "rel_decode_b4_k16384", b=4, h=32, sq=1, sk=16384, d=128, bidirectional=False),
        # A training step of an encoder layer at the usual length, padded sequences.
        _attn("train", "rel_train_s512_padded", b=16, h=12, sq=512, sk=512, d=64, padded=True),
        # A training step of a decoder layer at a 4k context: the largest backward here.
        _attn("train", "rel_train_s4096_d128", b=2, h=16, sq=4096, sk=4096, d=128, bidirectional=False, causal=True),
        # Ragged lengths, a head_dim between the kernels' own, fp16, many buckets over far distances.
        _attn("train", "rel_train_ragged_d80", b=2, h=12, sq=1000, sk=1531, d=80, dtype="f16", buckets=64,
              distance=640),
        # The gradients of a GPT-2-medium-shaped list in fp32, for clipping or for the training log.
        _list("norm", "norm_gpt2_medium_f32", shapes="gpt2_medium", param="f32"),
        # The reference's smallest optimizer benchmark point: the launches themselves count.
        _list("norm", "norm_8192_bf16", shapes="spread", param="bf16", tensors=1, smallest=8192, largest=8192),
        # The clipped optimizer step of a GPT-2-medium-shaped list: fp32 weights, bf16 momentum.
        _list("lion", "lion_clip_gpt2_medium", shapes="gpt2_medium", param="f32", momentum="bf16"),
        # The clipped step of a small all-bf16 list of adapter-sized tensors.
        _list("lion", "lion_clip_adapters_bf16", shapes="spread", param="bf16", momentum="bf16", tensors=48,
              smallest=768, largest=262_144),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _length(rng, lo, hi):
    """A sequence length: half of them multiples of 64, half any number."""
    n = _log_int(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    pick = rng.random()
    if pick < 0.3:
        while True:
            tensors = _log_int(rng, 1, 300)
            smallest = _log_int(rng, 8, 1_000_000)
            largest = max(smallest, _log_int(rng, 1024, 16_000_000))
            param, momentum = rng.choice([("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
            case = _list("norm" if pick < 0.12 else "lion", shapes="spread", param=param, momentum=momentum,
                         tensors=tensors, smallest=smallest, largest=largest)
            if sum(math.prod(s) for s in _shapes(case)) <= NUMEL_MOST:
                return case
    d = rng.choice([64, 64, 128, 128, 32, 40, 80, 96])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    h = rng.choice([4, 8, 12, 16, 32])
    # what keeps the logarithmic buckets apart: at least one distance for each of them
    buckets = rng.choice([16, 32, 32, 32, 64])
    distance = buckets * rng.choice([2, 4, 4, 10, 32])
    if pick < 0.45:
        b = _log_int(rng, 1, 32)
        sk = _length(rng, 64, max(65, min(32768, 16_000_000 // (b * h * 2))))
        return _attn("fwd", b=b, h=h, sq=1, sk=sk, d=d, dtype=dtype, buckets=buckets, distance=distance,
                     bidirectional=False, padded=rng.random() < 0.3)
    kind, most = ("fwd", FWD_SCORES_MOST) if pick < 0.7 else ("train", TRAIN_SCORES_MOST)
    while True:
        b = _log_int(rng, 1, 32)
        sq = _length(rng, 64, 8192)
        causal = rng.random() < 0.5
        sk = sq if causal or rng.random() < 0.6 else _length(rng, 64, 8192)
        if b * h * sq * sk <= most:
            return _attn(kind, b=b, h=h, sq=sq, sk=sk, d=d, dtype=dtype, buckets=buckets, distance=distance,
                         bidirectional=not causal, causal=causal, padded=not causal and rng.random() < 0.4)


# ---- inputs --------------------------------------------------------------------------------------

def _shapes(case):
    if case["shapes"] == "gpt2_medium":
        c = 1024
        block = [(c, 3 * c), (3 * c,), (c, c), (c,), (c, 4 * c), (4 * c,), (4 * c, c), (c,), (c,), (c,), (c,), (c,)]
        return [(50257, c), (1024, c)] + block * 24 + [(c,), (c,)]
    n, lo, hi = case["tensors"], case["smallest"], case["largest"]
    shapes = []
    for i in range(n):  # spread over the logarithm, in no sorted order
        t = ((i * 0.6180339887498949) % 1.0) if n > 1 else 0.0
        shapes.append((int(round(lo * (hi / lo) ** t)),))
    return shapes


def _prepare_list(case, seed):
    """Parameters, gradients and momentum as views of one buffer each (flat parameter storage,
    gradient buckets), every tensor on a 512-byte boundary as the caching allocator places them; the
    elements between the tensors are zeros.  The gradients' norm is several times `max_norm`, so that the
    step has to clip."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pdt, mdt = DTYPES[case["param"]], DTYPES[case["momentum"]]
    shapes = _shapes(case)
    offsets, at = [], 0
    for s in shapes:
        offsets.append(at)
        at += (math.prod(s) + 255) // 256 * 256
    numel = sum(math.prod(s) for s in shapes)
    flat_g = torch.empty(at, dtype=pdt, device="cuda").normal_(0.0, 1e-3, generator=gen)
    for s, o in zip(shapes, offsets):
        flat_g[o + math.prod(s):o + (math.prod(s) + 255) // 256 * 256] = 0
    grads = [flat_g[o:o + math.prod(s)].view(s) for s, o in zip(shapes, offsets)]
    state = {"kind": case["kind"], "grads": grads, "flat_g": flat_g}
    if case["kind"] == "norm":
        return state
    flat_p = torch.empty(at, dtype=pdt, device="cuda").normal_(0.0, 0.02, generator=gen)
    flat_m = torch.empty(at, dtype=mdt, device="cuda").normal_(0.0, 5e-4, generator=gen)
    for s, o in zip(shapes, offsets):
        flat_p[o + math.prod(s):o + (math.prod(s) + 255) // 256 * 256] = 0
        flat_m[o + math.prod(s):o + (math.prod(s) + 255) // 256 * 256] = 0
    state |= {"flat_p": flat_p, "flat_m": flat_m, "lr": 1e-4, "weight_decay": 0.1,
              "max_norm": 0.25e-3 * math.sqrt(numel)}
    if own:
        from fast_ops_b200.lion import Lion

        params = []
        for s, o, g in zip(shapes, offsets, grads):
            p = torch.nn.Parameter(flat_p[o:o + math.prod(s)].view(s))
            p.grad = g
            params.append(p)
        opt = Lion(params, lr=state["lr"], betas=BETAS, weight_decay=state["weight_decay"], momentum_dtype=mdt,
                   max_grad_norm=state["max_norm"])
        for p, o in zip(params, offsets):
            opt.state[p]["exp_avg"] = flat_m[o:o + p.numel()].view(p.shape)
        state["opt"] = opt
    return state


def _prepare_attn(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    b, h, sq, sk, d = (case[k] for k in ("b", "h", "sq", "sk", "d"))

    def tensor(*shape, std=1.0):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(0.0, std, generator=gen)

    state = {"kind": case["kind"], "q": tensor(b, h, sq, d), "k": tensor(b, h, sk, d), "v": tensor(b, h, sk, d),
             "table": tensor(case["buckets"], h, std=0.5), "distance": case["distance"],
             "bidirectional": case["bidirectional"], "causal": case["causal"],
             "offset": sk - 1 if sq == 1 else 0, "bias": None}
    if case["kind"] == "train":
        state["grad_out"] = tensor(b, h, sq, d)
        for name in ("q", "k", "v", "table"):
            state[name].requires_grad_()
    if case["padded"]:  # the last few keys of each sequence are masked
        lens = sk - torch.randint(0, max(1, sk // 4), (b, 1), generator=gen, device="cuda")
        keys = torch.arange(sk, device="cuda")
        state["bias"] = torch.zeros(b, sk, device="cuda").masked_fill(keys >= lens, float("-inf")).view(b, 1, 1, sk)
    return state


def prepare(case, seed):
    return _prepare_attn(case, seed) if case["kind"] in ("fwd", "train") else _prepare_list(case, seed)


# ---- the plain forms -----------------------------------------------------------------------------

def _buckets(distance_to_key, buckets, most, bidirectional):
    """Bucket of each relative position (key minus query): one for each of the nearest, then evenly
    spaced in the logarithm up to `most`.  The logarithm is taken in 64 bits, and a distance that lies
    on a border belongs to the farther bucket."""
    half = buckets // 2 if bidirectional else buckets
    near = half // 2
    n = distance_to_key.abs() if bidirectional else (-distance_to_key).clamp(min=0)
    far = torch.log(n.clamp(min=1).double() / near) / math.log(most / near) * (half - near)
    far = (near + torch.floor(far + 1e-9).long()).clamp(max=half - 1)
    side = (distance_to_key > 0).long() * half if bidirectional else 0
    return torch.where(n < near, n, far) + side


def _diagonals(sq, sk, offset, device):
    """Relative positions of the diagonals, from that of the last query and the first key on."""
    return torch.arange(1 - sq, sk, device=device) - offset


def _plain_attention(state):
    """(O, P, scale) in 32 bits; P (B, H, Sq, Sk)."""
    q, k, v, table = (state[name].detach().float() for name in ("q", "k", "v", "table"))
    sq, sk = q.shape[2], k.shape[2]
    ids = _buckets(_diagonals(sq, sk, state["offset"], q.device), table.shape[0], state["distance"],
                   state["bidirectional"])
    rows, cols = torch.arange(sq, device=q.device)[:, None], torch.arange(sk, device=q.device)[None, :]
    scale = 1.0 / math.sqrt(q.shape[3])
    s = q @ k.transpose(2, 3)
    s.mul_(scale)
    s += table[ids].T.contiguous()[:, cols - rows + sq - 1]
    if state["bias"] is not None:
        s += state["bias"]
    if state["causal"]:
        s.masked_fill_(cols > rows + state["offset"], float("-inf"))
    s -= s.amax(dim=-1, keepdim=True)
    p = s.exp_()
    p /= p.sum(dim=-1, keepdim=True)
    return p @ v, p, scale


def _plain_train(state):
    o, p, scale = _plain_attention(state)
    q, k, v, table, g = (state[name].detach().float() for name in ("q", "k", "v", "table", "grad_out"))
    sq, sk = q.shape[2], k.shape[2]
    dv = p.transpose(2, 3) @ g
    ds = g @ v.transpose(2, 3)
    ds -= (g * o).sum(dim=-1, keepdim=True)
    ds *= p
    dq = (ds @ k) * scale
    dk = (ds.transpose(2, 3) @ q) * scale
    # sums along the diagonals: rows in reverse order, each shifted by one against the one before
    skewed = torch.nn.functional.pad(ds.sum(dim=0).flip(1), (0, sq)).flatten(1)
    sums = skewed[:, :sq * (sk + sq - 1)].view(-1, sq, sk + sq - 1).double().sum(dim=1)
    ids = _buckets(_diagonals(sq, sk, state["offset"], q.device), table.shape[0], state["distance"],
                   state["bidirectional"])
    belongs = ids[None, :] == torch.arange(table.shape[0], device=q.device)[:, None]
    dtable = belongs.double() @ sums.T
    dt = state["q"].dtype
    return o.to(dt), dq.to(dt), dk.to(dt), dv.to(dt), dtable.to(dt)


def _plain_norm(state):
    return state["flat_g"].double().square_().sum().sqrt().float()


def _plain_lion(state):
    """The step is defined rounding by rounding (every product and sum is rounded to the type of the tensor
    that holds it), so the plain form rounds in the same places, between operations in 32 bits."""
    p, g, m = state["flat_p"], state["flat_g"], state["flat_m"]
    lr, wd, (b1, b2) = state["lr"], state["weight_decay"], BETAS
    norm = _plain_norm(state)
    coef = (norm.new_full((), state["max_norm"]) / (norm + 1e-6)).clamp(max=1.0)
    both = p.dtype if p.dtype == m.dtype else torch.float32
    g = (g.float() * coef).to(g.dtype).float()
    u = ((m.float() * b1).to(m.dtype).float() + (g * (1 - b1)).to(p.dtype).float()).to(both)
    step = norm.new_full((), lr).to(both).float()
    p.copy_((p.float() * (1 - lr * wd)).to(p.dtype).float() - step * u.float().sign())
    share = norm.new_full((), 1 - b2).to(both).float()
    # one rounding for product and sum: exact in 64 bits up to the last
    m.copy_(((m.float() * b2).to(m.dtype).double() + share.double() * g.double()).float())
    return p, m, norm


# ---- one pass ------------------------------------------------------------------------------------

def _own_attention(state):
    from fast_ops_b200.flash_attention import relative_attention

    return relative_attention(state["q"], state["k"], state["v"], state["table"], max_distance=state["distance"],
                              bidirectional=state["bidirectional"], query_offset=state["offset"],
                              causal=state["causal"], bias=state["bias"])


def run(state):
    kind = state["kind"]
    if not own:
        if kind == "fwd":
            return _plain_attention(state)[0].to(state["q"].dtype)
        return {"train": _plain_train, "norm": _plain_norm, "lion": _plain_lion}[kind](state)
    if kind == "fwd":
        with torch.no_grad():
            return _own_attention(state)
    if kind == "train":
        o = _own_attention(state)
        inputs = (state["q"], state["k"], state["v"], state["table"])
        return (o, *torch.autograd.grad(o, inputs, state["grad_out"]))
    if kind == "norm":
        from fast_ops_b200.lion import grad_norm

        return grad_norm(state["grads"])
    state["opt"].step()
    return state["flat_p"], state["flat_m"], state["opt"].grad_norm


# ---- in 64 bits ----------------------------------------------------------------------------------

def _borders(buckets, most, bidirectional):
    """Smallest distance of each logarithmic bucket after the first, from whole numbers alone: the bucket
    number near + x starts where (n / near)^(half - near) = (most / near)^x."""
    half = buckets // 2 if bidirectional else buckets
    near = half // 2
    w = half - near
    found, n = [], near
    for x in range(1, w):
        while n ** w * near ** x < most ** x * near ** w:
            n += 1
        found.append(n)
    return half, near, found


def _exact_attention(case, seed):
    state = _prepare_attn(case, seed)
    train = case["kind"] == "train"
    q, k, v, table = (state[name].detach() for name in ("q", "k", "v", "table"))
    b, h, sq, sk, d = (case[name] for name in ("b", "h", "sq", "sk", "d"))
    half, near, borders = _borders(case["buckets"], case["distance"], case["bidirectional"])
    delta = (torch.arange(sk, device=q.device)[None, :] - torch.arange(sq, device=q.device)[:, None]
             - state["offset"])
    n = delta.abs() if case["bidirectional"] else (-delta).clamp(min=0)
    ids = n.clamp(max=near)
    for border in borders:
        ids += n >= border
    if case["bidirectional"]:
        ids += half * (delta > 0)
    hidden = delta > 0 if case["causal"] else None
    o = torch.empty(b, h, sq, d, dtype=torch.float64, device=q.device)
    if train:
        dq, dk, dv = torch.empty_like(o), torch.empty_like(k, dtype=torch.float64), torch.empty_like(v, dtype=torch.float64)
        dtable = torch.zeros(case["buckets"], h, dtype=torch.float64, device=q.device)
    for i in range(b):
        for j in range(h):
            s = q[i, j].double() @ k[i, j].double().T / math.sqrt(d) + table[:, j].double()[ids]
            if state["bias"] is not None:
                s += state["bias"][i, 0].double()
            if hidden is not None:
                s.masked_fill_(hidden, float("-inf"))
            p = torch.softmax(s, dim=-1)
            o[i, j] = p @ v[i, j].double()
            if not train:
                continue
            g = state["grad_out"][i, j].double()
            ds = p * (g @ v[i, j].double().T - (g * o[i, j]).sum(-1, keepdim=True))
            dv[i, j] = p.T @ g
            dq[i, j] = ds @ k[i, j].double() / math.sqrt(d)
            dk[i, j] = ds.T @ q[i, j].double() / math.sqrt(d)
            for u in range(case["buckets"]):
                dtable[u, j] += (ds * (ids == u)).sum()
    return (o, dq, dk, dv, dtable) if train else o


def _exact_lion(case, seed):
    """Which way an element moves is decided by terms that are rounded to the types of gradient and momentum
    by the step's definition; everything else in 64 bits."""
    state = _prepare_list(case, seed)
    (pdt, mdt), (b1, b2) = (DTYPES[case["param"]], DTYPES[case["momentum"]]), BETAS
    p, g, m = state["flat_p"].double(), state["flat_g"].double(), state["flat_m"].double()
    norm = g.square().sum().sqrt()
    g = g * (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    u = (m * b1).to(mdt).double() + (g.to(pdt).double() * (1 - b1)).to(pdt).double()
    p = p * (1 - state["lr"] * state["weight_decay"]) - state["lr"] * u.sign()
    return p, m * b2 + g * (1 - b2), norm


def exact(case, seed):
    if case["kind"] == "norm":
        return _prepare_list(case, seed)["flat_g"].double().square().sum().sqrt()
    return _exact_lion(case, seed) if case["kind"] == "lion" else _exact_attention(case, seed)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["kind"] in ("norm", "lion"):
        n = sum(math.prod(s) for s in _shapes(case))
        e = SIZE[case["param"]]
        if case["kind"] == "norm":
            return {"bytes": n * e, "flops": 2.0 * n}
        # the norm needs every gradient before the first update: g read twice; p, m read and written
        return {"bytes": n * (4 * e + 2 * SIZE[case["momentum"]]), "flops": 14.0 * n}
    e = SIZE[case["dtype"]]
    b, h, sq, sk, d = (case[name] for name in ("b", "h", "sq", "sk", "d"))
    pairs = sq * sk
    if case["causal"]:
        pairs = sum(min(sk, i + 1) for i in range(sq))
    q, kv = b * h * sq * d * e, 2 * b * h * sk * d * e
    table = case["buckets"] * h * e
    moved = q + kv + table + (4 * b * sk if case["padded"] else 0) + q  # Q, K, V, table, mask in; O out
    flops = 4.0 * b * h * pairs * d
    if case["kind"] == "train":
        moved += q + q + kv + table  # dO in; dQ, dK, dV, dTable out
        flops *= 3.5                 # the backward's five matmuls against the forward's two
    return {"bytes": moved, "flops": flops}
