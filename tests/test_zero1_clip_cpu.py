"""Clipping by the global norm in the ZeRO-1 step: a world-size-2 gloo run on CPU in which the device calls (sum
of squares of a slice, norm and factor, step) are replaced by their formulas."""
import math
import os
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_zero1_cpu import ROOT, _free_port


def _worker(rank, world, port, reduce_gradients, ret):
    sys.path.insert(0, ROOT)
    import oracle
    from fast_ops_b200.lion import Lion

    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        gen = torch.Generator().manual_seed(7)
        shapes = [(33, 7), (1000,), (5,), (64, 64), (3,)]
        init = [(torch.randn(s, generator=gen) * 0.02).bfloat16() for s in shapes]
        params = [t.clone().requires_grad_(True) for t in init]
        opt = Lion(params, lr=1e-3, weight_decay=0.1, process_group=dist.group.WORLD, reduce_gradients=reduce_gradients,
                   max_grad_norm=0.05)
        zero = opt._zero
        calls = []

        def sumsq(flat_g, begin, end):
            calls.append((begin, end))
            return flat_g[begin:end].double().square().sum().reshape(1)

        def finish(total, max_norm):
            norm = total[0].sqrt().float()
            return norm, (torch.tensor(max_norm) / (norm + 1e-6)).clamp(max=1.0)

        def step(p, g, m_shard, begin, end, lr, betas, wd, clip=None):
            pp, gg = p[begin:end].clone(), (g[begin:end].float() * clip).to(g.dtype)
            oracle.lion_step(pp, gg, m_shard, lr, betas, wd)
            p[begin:end] = pp

        zero.sumsq_fn, zero.finish_norm_fn, zero.flat_step_fn = sumsq, finish, step
        ref_p, ref_m = [t.clone() for t in init], [torch.zeros_like(t) for t in init]
        for scale in (1.0, 1e-4):  # clipped, and not
            grads = [(torch.randn(s, generator=gen) * scale).to(torch.float8_e4m3fn).bfloat16() if scale == 1.0 else
                     (torch.randn(s, generator=gen).to(torch.float8_e4m3fn).bfloat16() * 2.0**-13) for s in shapes]
            for p, g in zip(params, grads):
                # the step averages these to g; 1.5 g needs a bit more than g, so g has bits to spare
                p.grad.copy_(g * (0.5 if rank == 0 else 1.5) if reduce_gradients else g)
            opt.step()
            want = math.sqrt(sum(g.double().square().sum().item() for g in grads))
            assert abs(opt.grad_norm.item() - want) <= 2.0**-23 * want
            coef = (torch.tensor(0.05) / (opt.grad_norm + 1e-6)).clamp(max=1.0)
            assert (coef < 1) == (scale == 1.0)
            for rp, g, rm in zip(ref_p, grads, ref_m):
                oracle.lion_step(rp.view(-1), (g.float() * coef).to(g.dtype).view(-1), rm.view(-1), 1e-3, (0.9, 0.99), 0.1)
            for p, rp in zip(params, ref_p):
                assert torch.equal(p.data, rp), f"rank {rank}: params differ"
        assert calls == [(zero.begin, zero.end)] * 2  # each rank sums its own slice only
        ret[rank] = "ok"
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("reduce_gradients", [False, True])
def test_clipping_over_two_ranks(reduce_gradients):
    ret = mp.Manager().dict()
    mp.spawn(_worker, args=(2, _free_port(), reduce_gradients, ret), nprocs=2, join=True)
    assert dict(ret) == {0: "ok", 1: "ok"}
