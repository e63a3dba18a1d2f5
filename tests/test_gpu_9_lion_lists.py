"""Lion steps after the optimizer's tensors were exchanged between two of them: bit for bit the step of a new
optimizer that is given the tensors as they are then."""
import pytest
import torch

from fast_ops_b200.lion import Lion, grad_norm

pytestmark = pytest.mark.gpu
OPTIONS = dict(lr=1e-3, weight_decay=0.1)


def build(shapes, max_norm, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(len(shapes))
    params = [torch.nn.Parameter(torch.empty(s, device="cuda").normal_(0, 0.02, generator=gen).to(dtype)) for s in shapes]
    for p in params:
        p.grad = torch.empty(p.shape, device="cuda").normal_(0, 1e-2, generator=gen).to(dtype)
    return params, Lion(params, **OPTIONS, max_grad_norm=max_norm)


def step_and_compare(params, opt):
    twins = [torch.nn.Parameter(p.detach().clone(memory_format=torch.preserve_format)) for p in params]
    ref = Lion(twins, **OPTIONS, max_grad_norm=opt.max_grad_norm)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone(memory_format=torch.preserve_format)
        if "exp_avg" in opt.state.get(p, {}):
            ref.state[q]["exp_avg"] = opt.state[p]["exp_avg"].clone()
    opt.step()
    ref.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert torch.equal(opt.state[p]["exp_avg"], ref.state[q]["exp_avg"])
    if opt.max_grad_norm is not None:
        assert torch.equal(opt.grad_norm, ref.grad_norm)
        assert torch.equal(opt.grad_norm, grad_norm([p.grad for p in params]))


@pytest.mark.parametrize("max_norm", [None, 0.05])
@pytest.mark.parametrize("shapes", [[(5000,)], [(5000,), (33, 70), (9000,)]])
def test_exchanged_momentum(shapes, max_norm, cuda_device):
    params, opt = build(shapes, max_norm)
    step_and_compare(params, opt)
    opt.state[params[0]]["exp_avg"] = torch.full_like(params[0], 0.25)
    step_and_compare(params, opt)
    for p in params:  # the tensors before are freed
        opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"].float()
    step_and_compare(params, opt)
    assert all(opt.state[p]["exp_avg"].dtype == torch.float32 for p in params)
    for p in params:  # away and back again
        opt.state[p]["exp_avg"].data = opt.state[p]["exp_avg"].cpu()
    blocker = [torch.full_like(p, 7.0, dtype=torch.float32) for p in params]
    for p in params:
        opt.state[p]["exp_avg"].data = opt.state[p]["exp_avg"].cuda()
    step_and_compare(params, opt)
    opt.state.clear()
    step_and_compare(params, opt)
    assert all((b == 7.0).all() for b in blocker)


@pytest.mark.parametrize("max_norm", [None, 0.05])
def test_shortened_and_transposed_tensors(max_norm, cuda_device):
    params, opt = build([(5000,), (64, 64), (9000,)], max_norm)
    step_and_compare(params, opt)
    p, rest = params[0], params[0].detach()[100:].clone()
    whole, momentum = p.detach(), opt.state[p]["exp_avg"]
    rest_momentum = momentum[100:].clone()
    p.data = p.data[:100]
    p.grad = p.grad[:100]
    with pytest.raises(RuntimeError):
        opt.step()
    opt.state[p]["exp_avg"] = momentum[:100]
    step_and_compare(params, opt)
    assert torch.equal(whole[100:], rest) and torch.equal(momentum[100:], rest_momentum)
    q = params[1]
    q.grad = q.grad.t()
    with pytest.raises(RuntimeError):
        opt.step()


@pytest.mark.parametrize("max_norm", [None, 0.05])
def test_new_gradients_every_step(max_norm, cuda_device):
    params, opt = build([(5000,), (64, 64), (9000,)], max_norm)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(4):
        opt.zero_grad(set_to_none=True)
        for p in params:
            p.grad = torch.empty_like(p).normal_(0, 1e-2, generator=gen)
        step_and_compare(params, opt)
