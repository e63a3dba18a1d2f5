"""The global gradient norm and the Lion step that clips by it.

Norm: the sum is formed in double from fp32 sums of eight squares (relative error below 7 half steps of fp32
each), the result is rounded to fp32 once: at most (7 / 2 + 1) * 2^-24 relative to the norm in 64 bits.
Clipped step: bit for bit the step of gradients that were clipped in memory, round(g * coef) with
coef = min(1, max_norm / (norm + 1e-6)) in fp32, for the norm that the call reports.
"""
import math

import pytest
import torch

import oracle
from fast_ops_b200 import _lib as L
from fast_ops_b200.lion import Lion, grad_norm
from fast_ops_b200.lion.lion_optimizer import _flat_step, _flat_step_push

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
NORM_TOL = 4.5 * 2.0**-24


def norm64(ts):
    return math.sqrt(sum(t.detach().double().square().sum().item() for t in ts))


def randoms(shapes, dtypes, seed=0, std=1e-2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.empty(s, device="cuda").normal_(0, std, generator=gen).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(shapes)]


@pytest.mark.parametrize("dtypes", [(FP,), (BF,), (HF,), (FP, BF, HF)])
@pytest.mark.parametrize("shapes", [
    [(1,)], [(8192,)], [(8193,)], [(7,), (0,), (3, 5), (4097,), (12345,)], [(0,), (0,)], [(1 << 20,), (33,)],
    [(5000,)] * 32, [(5000,)] * 33, [(1 << 18,)], [((1 << 18) + 1,)], [(257,)] * 95, [(31,)] * 96, [(1000 + i,) for i in range(97)], [(64,)] * 1024, [(5 + i % 7,) for i in range(2500)],
])
def test_norm_matches_64_bits(shapes, dtypes, cuda_device):
    gs = randoms(shapes, dtypes, seed=len(shapes))
    got = grad_norm(gs)
    assert got.shape == () and got.dtype == FP and got.device == gs[0].device
    want = norm64(gs)
    assert abs(got.item() - want) <= NORM_TOL * want
    assert torch.equal(got, grad_norm(gs))  # the same bits again


def test_norm_of_unaligned_transposed_and_single_tensors(cuda_device):
    base = randoms([(100_003,)], (BF,))[0]
    for cut in (base[1:], base[3:9000], base[5:]):
        want = norm64([cut])
        assert abs(grad_norm([cut]).item() - want) <= NORM_TOL * want
    t = randoms([(300, 77)], (FP,))[0]
    assert abs(grad_norm(t.T).item() - norm64([t])) <= NORM_TOL * norm64([t])
    assert torch.equal(grad_norm(iter([t, base])), grad_norm([t, base]))
    assert not grad_norm([t.requires_grad_()]).requires_grad


@pytest.mark.parametrize("value", [1e30, 3e38, 1e-30, 1e-42, 0.0])
def test_norm_of_values_whose_squares_leave_fp32(value, cuda_device):
    g = torch.full((20_000,), value, device="cuda")
    want = norm64([g])
    got = grad_norm([g]).item()
    if want > torch.finfo(FP).max:
        assert got == math.inf
    else:
        # below the normal numbers of fp32 the result itself is rounded to 2^-149
        assert abs(got - want) <= max(NORM_TOL * want, 2.0**-150)
    mixed = torch.cat([g, torch.full((7,), 2.0, device="cuda")])
    if value < 1e30:
        assert abs(grad_norm([mixed]).item() - math.sqrt(28)) <= NORM_TOL * math.sqrt(28)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [0, 8191, 8192, 9000])
@pytest.mark.parametrize("dtype", [FP, BF, HF])
def test_non_finite_gradients_show(bad, at, dtype, cuda_device):
    g = torch.ones(9001, device="cuda", dtype=dtype)
    g[at] = bad
    got = grad_norm([g]).item()
    assert math.isnan(got) if math.isnan(bad) else got == math.inf


def test_a_tensor_beyond_32_bit_element_counts(cuda_device):
    g = torch.zeros((1 << 31) + 12345, device="cuda", dtype=BF)
    g[-1], g[1 << 31], g[0] = 3.0, 4.0, 12.0
    assert grad_norm([g]).item() == 13.0


def test_norm_in_a_graph_and_on_another_stream(cuda_device):
    gs = randoms([(5000,), (70_000,)], (FP, BF))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # no call outside before it
        n = grad_norm(gs)
    for g in gs:
        g.mul_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(n, grad_norm(gs))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m = grad_norm(gs)
    side.synchronize()
    assert torch.equal(n, m)


def test_norm_refusals(cuda_device):
    t = torch.ones(8, device="cuda")
    for bad in ([], [t.cpu()], [t, t.cpu()], [t.double()], [t[::2]], [t.expand(3, 8)], [t.to_sparse()], [1.0],
                [t.to(torch.complex64)]):
        with pytest.raises(RuntimeError):
            grad_norm(bad)


# ---- the clipped step ----------------------------------------------------------------------------

def clipped(g, norm, max_norm):
    coef = (torch.full((), max_norm, device=norm.device) / (norm + 1e-6)).clamp(max=1.0)
    return (g.float() * coef).to(g.dtype)


def problem(shapes, pdt, mdt, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda s, std, dt: torch.empty(s, device="cuda").normal_(0, std, generator=gen).to(dt)  # noqa: E731
    return [r(s, 0.02, pdt) for s in shapes], [r(s, 1e-3, pdt) for s in shapes], [r(s, 5e-4, mdt) for s in shapes]


SHAPES = [(4097,), (3, 5), (50000,), (8,), (1 << 18,), (12345,)]


@pytest.mark.parametrize("pdt,mdt", [(BF, BF), (BF, FP), (BF, HF), (HF, HF), (HF, FP), (HF, BF), (FP, FP), (FP, BF), (FP, HF)])
@pytest.mark.parametrize("shapes", [SHAPES, SHAPES[:1], SHAPES[4:5]])
@pytest.mark.parametrize("share", [0.1, 3.0])  # max_norm over the norm: clips, does not
def test_clipped_step_is_the_step_of_clipped_gradients(pdt, mdt, shapes, share, cuda_device):
    ps, gs, ms = problem(shapes, pdt, mdt, seed=3)
    max_norm = share * norm64(gs)
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    for p, g in zip(params, gs):
        p.grad = g.clone()
    opt = Lion(params, lr=1e-3, weight_decay=0.1, momentum_dtype=mdt, max_grad_norm=max_norm)
    for p, m in zip(params, ms):
        opt.state[p]["exp_avg"] = m.clone()
    plain = [torch.nn.Parameter(p.clone()) for p in ps]
    ref = Lion(plain, lr=1e-3, weight_decay=0.1, momentum_dtype=mdt)
    for p, m in zip(plain, ms):
        ref.state[p]["exp_avg"] = m.clone()
    for _ in range(2):  # the momentum of the first step feeds the second
        opt.step()
        assert abs(opt.grad_norm.item() - norm64(gs)) <= NORM_TOL * norm64(gs)
        for p, g in zip(plain, gs):
            p.grad = clipped(g, opt.grad_norm, max_norm)
        ref.step()
    for p, q, g in zip(params, plain, gs):
        assert torch.equal(p, q)
        assert torch.equal(opt.state[p]["exp_avg"], ref.state[q]["exp_avg"])
        assert torch.equal(p.grad, g)  # the stored gradient is left as it is


def test_clipped_step_against_the_cpu_oracle(cuda_device):
    ps, gs, ms = problem([(9000,), (77,)], BF, BF, seed=11)
    params = [torch.nn.Parameter(p.clone()) for p in ps]
    for p, g in zip(params, gs):
        p.grad = g
    opt = Lion(params, lr=1e-3, weight_decay=0.1, max_grad_norm=0.01)
    for p, m in zip(params, ms):
        opt.state[p]["exp_avg"] = m.clone()
    opt.step()
    for p, p0, g, m0 in zip(params, ps, gs, ms):
        rp, rg, rm = p0.cpu(), clipped(g, opt.grad_norm, 0.01).cpu(), m0.cpu()
        oracle.lion_step(rp, rg, rm, 1e-3, (0.9, 0.99), 0.1)
        assert torch.equal(p.detach().cpu(), rp) and torch.equal(opt.state[p]["exp_avg"].cpu(), rm)


def test_the_norm_runs_over_all_groups_and_types(cuda_device):
    a = [torch.nn.Parameter(torch.zeros(100, device="cuda", dtype=BF)), torch.nn.Parameter(torch.zeros(70, device="cuda"))]
    b = [torch.nn.Parameter(torch.zeros(33, device="cuda", dtype=BF)), torch.nn.Parameter(torch.zeros(9, device="cuda"))]
    a[0].grad, a[1].grad, b[0].grad = (torch.full_like(t, 2.0) for t in (a[0], a[1], b[0]))  # b[1] has none
    opt = Lion([{"params": a, "lr": 1e-3}, {"params": b, "lr": 1e-2}], max_grad_norm=1.0)
    assert opt.grad_norm is None
    opt.step()
    first = opt.grad_norm
    assert abs(first.item() - 2 * math.sqrt(203)) <= NORM_TOL * 2 * math.sqrt(203)
    b[1].grad = torch.full_like(b[1], 2.0)
    opt.step()
    assert abs(opt.grad_norm.item() - 2 * math.sqrt(212)) <= NORM_TOL * 2 * math.sqrt(212)
    assert abs(first.item() - 2 * math.sqrt(203)) <= NORM_TOL * 2 * math.sqrt(203)  # a norm kept is not overwritten
    assert (a[0] < 0).all() and torch.equal(b[1], torch.full_like(b[1], -1e-2))
    for t in a + b:
        t.grad = None
    before = [t.detach().clone() for t in a + b]
    opt.step()
    assert opt.grad_norm is None and all(torch.equal(x, y) for x, y in zip(before, a + b))


def test_clipping_options(cuda_device):
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(RuntimeError):
            Lion([p], max_grad_norm=bad)
    p.grad = torch.ones_like(p)
    opt = Lion([p], lr=1e-3, max_grad_norm=math.inf)  # the norm alone
    opt.step()
    assert torch.equal(opt.state[p]["exp_avg"], torch.full_like(p, 0.01))
    opt.max_grad_norm = 0.5 * math.sqrt(10)
    opt.state[p]["exp_avg"].zero_()
    opt.step()
    coef = (torch.full((), 0.5 * math.sqrt(10), device="cuda") / (opt.grad_norm + 1e-6)).item()
    assert torch.allclose(opt.state[p]["exp_avg"], torch.full_like(p, 0.01 * coef), rtol=2.0**-22, atol=0)
    opt.max_grad_norm = -1.0
    with pytest.raises(RuntimeError):
        opt.step()


def test_no_norm_is_left_from_a_step_before_clipping_was_turned_off(cuda_device):
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = Lion([p], max_grad_norm=1.0)
    opt.step()
    assert opt.grad_norm.item() == torch.tensor(10.0).sqrt().item()
    opt.max_grad_norm = None
    opt.step()
    assert opt.grad_norm is None


def test_a_gradient_of_infinities_does_not_pass_for_a_small_one(cuda_device):
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    p.grad = torch.full_like(p, 1.0)
    p.grad[3] = math.inf
    opt = Lion([p], lr=1e-3, max_grad_norm=1.0)
    opt.step()
    assert opt.grad_norm.item() == math.inf
    # coef is 0: finite gradients vanish, the infinite one gives NaN
    assert torch.isnan(opt.state[p]["exp_avg"][3]) and (opt.state[p]["exp_avg"][:3] == 0).all()


def test_clipped_step_in_a_graph(cuda_device):
    ps, gs, ms = problem(SHAPES, FP, BF, seed=5)

    def build():
        params = [torch.nn.Parameter(p.clone()) for p in ps]
        for p, g in zip(params, gs):
            p.grad = g.clone()
        opt = Lion(params, lr=1e-3, weight_decay=0.1, momentum_dtype=BF, max_grad_norm=0.05)
        return params, opt

    (pa, a), (pb, b) = build(), build()
    a.step()  # outside the capture: the step's tensor table is made
    b.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.step()
    for p, q in zip(pa, pb):
        p.grad.mul_(0.7)
        q.grad.mul_(0.7)
    for _ in range(2):
        graph.replay()
        b.step()
    torch.cuda.synchronize()
    assert torch.equal(a.grad_norm, b.grad_norm)
    for p, q in zip(pa, pb):
        assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])


@pytest.mark.parametrize("step", ["flat", "push"])
def test_clipped_flat_steps(step, cuda_device):
    """The shard forms of the ZeRO-1 step (the peer-store one without peers)."""
    n, begin, end = 100_000, 1000, 90_008
    (p,), (g,), (m,) = problem([(n,)], BF, BF, seed=2)
    m = m[begin:end].clone()
    clip = torch.tensor([0.25], device="cuda")
    p2, m2 = p.clone(), m.clone()
    args = (1e-3, (0.9, 0.99), 0.1)
    if step == "flat":
        _flat_step(p, g, m, begin, end, *args, clip=clip)
    else:
        _flat_step_push(p, g, m, begin, end, [], *args, clip=clip)
    _flat_step(p2, (g.float() * 0.25).to(BF), m2, begin, end, *args)
    assert torch.equal(p, p2) and torch.equal(m, m2)


def test_refused_entry_arguments(cuda_device):
    import ctypes

    lib = L.load()
    t = torch.ones(8, device="cuda")
    ptr, num, dt = (ctypes.c_void_p * 1)(t.data_ptr()), (ctypes.c_int64 * 1)(8), (ctypes.c_int * 1)(L.FO_F32)
    ws = torch.empty(lib.fo_grad_norm_workspace(1), dtype=torch.float64, device="cuda")
    out = torch.empty(2, device="cuda")
    ok = (ptr, num, dt, 1, 1.0, ws.data_ptr(), None, out.data_ptr(), out.data_ptr() + 4, 0, None)

    def with_(i, v):
        a = list(ok)
        a[i] = v
        return lib.fo_grad_norm(*a)

    assert lib.fo_grad_norm(*ok) == 0
    for i, v in ((3, -1), (4, -1.0), (4, math.nan), (5, None), (0, (ctypes.c_void_p * 1)(None)),
                 (1, (ctypes.c_int64 * 1)(-1)), (2, (ctypes.c_int * 1)(7)), (0, (ctypes.c_void_p * 1)(t.data_ptr() + 2)),
                 (5, ws.data_ptr() + 4)):
        assert with_(i, v) == -1, i
    assert lib.fo_grad_norm(ptr, num, dt, 1, 1.0, ws.data_ptr(), None, None, None, 0, None) == -1
    for args in ((None, 1.0, out.data_ptr(), None), (ws.data_ptr(), 1.0, None, None), (ws.data_ptr(), -1.0, out.data_ptr(), None)):
        assert lib.fo_grad_norm_finish(*args, 0, None) == -1
    torch.cuda.synchronize()
    assert out[0].item() == pytest.approx(math.sqrt(8), rel=1e-6) and out[1].item() == pytest.approx(1 / math.sqrt(8), rel=1e-6)
