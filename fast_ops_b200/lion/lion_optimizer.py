"""Fused Lion optimizer with the reference's torch.optim interface.

Mirrors fast_ops/lion/lion_optimizer.py of jfc4050/fast-ops (`Lion.__init__` :34-55, `step`
:57-76): same constructor defaults, `RuntimeError` on a non-positive learning rate or a beta
outside [0, 1], state key "exp_avg", param-group keys lr / betas / weight_decay.  Instead of
one kernel launch per tensor, `step()` hands every (param, grad, exp_avg) triple of a group to
ONE multi-tensor kernel launch per dtype combination.  The arithmetic follows the reference
torch implementation (fast_ops/lion/lion_optimizer_ref.py:51-67) rounding for rounding.

Keyword-only extensions:
  momentum_dtype   dtype of exp_avg (default: the parameter's dtype, as the reference does at
                   :68-74; the Lion paper keeps momentum in bf16).
  process_group    a torch.distributed group: parameters are laid out in one flat buffer, each
                   rank updates only its 1/world_size slice (and keeps momentum only for it),
                   then ONE all-gather distributes the updated weights (ZeRO-1).
  fused_gather     with process_group: the flat parameter buffer is a symmetric-memory
                   allocation and the step kernel itself stores the updated slice into every
                   peer's buffer over NVLink, replacing the all-gather.
  reduce_gradients with process_group: step() first averages the flat gradient buffer across
                   the ranks with one reduce-scatter into this rank's slice (otherwise the caller
                   is expected to have reduced the gradients already).
  max_grad_norm    step() first takes the 2-norm over the gradients of all parameters (over all
                   ranks' slices with process_group) and applies every gradient times
                   min(1, max_grad_norm / (norm + 1e-6)), rounded to the gradient's type once, as if
                   it had been clipped in memory.  The factor stays on the device and the stored
                   gradients are left as they are.  `grad_norm` is the norm of the latest step.  A NaN
                   among the gradients makes the factor NaN, an infinity makes it 0 (finite gradients
                   vanish, infinite ones give NaN); finite gradients whose norm is beyond fp32 are
                   scaled by that norm, though `grad_norm` is infinite.
"""
from __future__ import annotations

import ctypes
from itertools import repeat
from operator import attrgetter, call, is_
from typing import Dict, Iterable, List, Optional, Tuple
from weakref import ref

import torch
from torch import Tensor
from torch.optim.optimizer import Optimizer

from .. import _lib
from .grad_norm import GradList, finish_norm, is_dense as _is_dense, shard_sumsq
from .zero1 import FlatLayout

_dtype_of = attrgetter("dtype")


def lion_update(param: Tensor, grad: Tensor, exp_avg: Tensor, lr: float, beta1: float, beta2: float,
                weight_decay: float) -> None:
    """Single-tensor fused step; the signature of the reference extension's `lion_update`
    (fast_ops/lion/lion.cpp:4-15).  Same checks as its host launcher
    (fast_ops/lion/lion_update.cu:132-139): param/grad dtypes equal, all three dense."""
    _check_triple(param, grad, exp_avg)
    lib = _lib.load()
    _lib.check(lib.fo_lion_update(
        param.data_ptr(), grad.data_ptr(), exp_avg.data_ptr(), param.numel(),
        _lib.dtype_code(param.dtype), _lib.dtype_code(grad.dtype), _lib.dtype_code(exp_avg.dtype),
        float(lr), float(beta1), float(beta2), float(weight_decay), param.device.index,
        _lib.current_stream_ptr(param.device)))


def _check_triple(param: Tensor, grad: Tensor, exp_avg: Tensor) -> None:
    if not param.is_cuda:
        raise RuntimeError("fast_ops_b200 Lion needs CUDA tensors (there is no CPU path)")
    if grad.device != param.device or exp_avg.device != param.device:
        raise RuntimeError("param, grad and exp_avg must be on the same device")
    if param.dtype != grad.dtype:
        raise RuntimeError(f"param and grad dtypes differ: {param.dtype} vs {grad.dtype}")
    if grad.shape != param.shape or exp_avg.numel() != param.numel():
        raise RuntimeError("param, grad and exp_avg must have the same number of elements")
    for t in (param, grad, exp_avg):
        if not _is_dense(t):
            raise RuntimeError("expected tensor to be contiguous")
    if param.stride() != grad.stride():
        raise RuntimeError("param and grad must share a memory layout")


def _flat_step_push(p: Tensor, g: Tensor, m_shard: Tensor, begin: int, end: int, peer_ptrs, lr: float, betas,
                    wd: float, clip: Optional[Tensor] = None) -> None:
    """Lion step on [begin, end) that also stores the result into the peers' flat buffers
    (C-ABI fo_lion_flat_step_push).  `peer_ptrs`: device addresses of the peers' element 0; `clip`: a
    device float that multiplies the gradients."""
    lib = _lib.load()
    n = len(peer_ptrs)
    arr = (ctypes.c_void_p * max(n, 1))(*peer_ptrs)
    entry, extra = (lib.fo_lion_flat_step_push, ()) if clip is None else (
        lib.fo_lion_flat_step_push_clipped, (clip.data_ptr(),))
    _lib.check(entry(
        p.data_ptr(), g.data_ptr(), m_shard.data_ptr(), begin, end, arr, n,
        _lib.dtype_code(p.dtype), _lib.dtype_code(g.dtype), _lib.dtype_code(m_shard.dtype),
        float(lr), float(betas[0]), float(betas[1]), float(wd), *extra, p.device.index,
        _lib.current_stream_ptr(p.device)))


def _flat_step(p: Tensor, g: Tensor, m_shard: Tensor, begin: int, end: int, lr: float, betas, wd: float,
               clip: Optional[Tensor] = None) -> None:
    """Lion step on elements [begin, end) of the flat buffers (C-ABI fo_lion_flat_step); `clip`: a device
    float that multiplies the gradients."""
    lib = _lib.load()
    entry, extra = (lib.fo_lion_flat_step, ()) if clip is None else (lib.fo_lion_flat_step_clipped, (clip.data_ptr(),))
    _lib.check(entry(
        p.data_ptr(), g.data_ptr(), m_shard.data_ptr(), begin, end,
        _lib.dtype_code(p.dtype), _lib.dtype_code(g.dtype), _lib.dtype_code(m_shard.dtype),
        float(lr), float(betas[0]), float(betas[1]), float(wd), *extra, p.device.index,
        _lib.current_stream_ptr(p.device)))


class _TensorList:
    """ctypes image of one multi-tensor call, issued again while `Lion._prepared` finds that it stands."""

    def __init__(self, key, params: List[Tensor], grads: List[Tensor], moms: List[Tensor]):
        n = len(params)
        _, self.device_index, p_dtype, m_dtype = key
        self.p_code, self.m_code = _lib.dtype_code(p_dtype), _lib.dtype_code(m_dtype)
        self.n = n
        self.params = (ctypes.c_void_p * n)(*[t.data_ptr() for t in params])
        self.grads = (ctypes.c_void_p * n)(*[t.data_ptr() for t in grads])
        self.moms = (ctypes.c_void_p * n)(*[t.data_ptr() for t in moms])
        self.numels = (ctypes.c_int64 * n)(*[t.numel() for t in params])


class Lion(Optimizer):
    """Lion ("Symbolic Discovery of Optimization Algorithms", arXiv:2302.06675), fused."""

    def __init__(self, params: Iterable, lr: float = 1e-4, betas: Tuple[float, float] = (0.9, 0.99),
                 weight_decay: float = 0.0, *, momentum_dtype: Optional[torch.dtype] = None,
                 process_group=None, fused_gather: bool = False, reduce_gradients: bool = False,
                 max_grad_norm: Optional[float] = None) -> None:
        if lr <= 0:
            raise RuntimeError(f"expected positive LR, got {lr}")
        if not all(0 <= beta <= 1 for beta in betas):
            raise RuntimeError(f"betas must be between 0 and 1. got {betas}")
        if momentum_dtype not in (None, torch.float16, torch.bfloat16, torch.float32):
            raise RuntimeError(f"unsupported momentum dtype {momentum_dtype}")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise RuntimeError(f"max_grad_norm must be positive, got {max_grad_norm}")
        defaults = {"lr": lr, "betas": betas, "weight_decay": weight_decay}
        super().__init__(params, defaults)
        self._momentum_dtype = momentum_dtype
        self._kept: Optional[tuple] = None  # what _prepared made for the step before
        self.max_grad_norm = max_grad_norm
        #: 0-d fp32 tensor: the norm of all gradients at the latest step, before clipping.  None before the
        #: first step, without max_grad_norm, and after a step in which no parameter had a gradient
        self.grad_norm: Optional[Tensor] = None
        self._grad_list: Optional[Tuple[list, Optional[GradList]]] = None
        self._pg = process_group
        self._zero = None
        if fused_gather and process_group is None:
            raise RuntimeError("fused_gather needs a process_group")
        if reduce_gradients and process_group is None:
            raise RuntimeError("reduce_gradients needs a process_group")
        if process_group is not None:
            self._zero = _Zero1State(self, process_group, momentum_dtype, fused_gather, reduce_gradients)

    # -- multi-tensor path ---------------------------------------------------------------
    # A training loop presents the same tensors step after step, so the checks and the pointer arrays of a step
    # stand for the next one.  They hold raw addresses, and an address alone says little: a view, or memory that the
    # allocator has given to another tensor, can have the one of the step before.  So a step first compares what they
    # were made from with the tensors it has now (0.4 us per parameter; new lists take 3 to 4).
    def _signature(self) -> Tuple[list, list]:
        """What the launches of a step are made from, column by column: the parameters of each group with their
        addresses, sizes and types; the addresses (None: no gradient) and strides of their gradients, which have the
        parameters' types and shapes (assigning others raises); the state's keys and its momentum tensors' addresses.
        Beside it the momentum tensors themselves, in the order of the state (None where there is none)."""
        groups = self.param_groups
        params = groups[0]["params"] if len(groups) == 1 else [p for group in groups for p in group["params"]]
        grads = [p.grad for p in params]
        try:
            momenta = list(map(dict.get, self.state.values(), repeat("exp_avg")))
            optional = [list(map(Tensor.data_ptr, grads)), list(map(Tensor.stride, grads)), list(map(Tensor.data_ptr, momenta))]
        except TypeError:  # a parameter without a gradient or a momentum, or something of the caller's own in the state
            momenta = [s.get("exp_avg") if isinstance(s, dict) else None for s in self.state.values()]
            optional = [[t if t is None else t.data_ptr() for t in grads], [t if t is None else t.stride() for t in grads],
                        [t if t is None else t.data_ptr() for t in momenta]]
        return [list(map(id, params)), list(map(Tensor.data_ptr, params)), list(map(Tensor.numel, params)),
                list(map(_dtype_of, params)), *optional, list(map(id, self.state)),
                [len(group["params"]) for group in groups]], momenta

    def _prepared(self) -> List[list]:
        """The launches of each group: those of the step before where they stand."""
        kept = self._kept
        if kept is not None:
            signature, momenta = self._signature()
            if kept[0] == signature and all(map(is_, map(call, kept[2]), momenta)):
                return kept[1]
        self._kept = None
        lists = [self._prepare_group(gi, group) for gi, group in enumerate(self.param_groups)]
        signature, momenta = self._signature()
        # A momentum tensor that the caller takes out of the state is to be freed, so it is held weakly; the
        # parameters and keys are held, so that their ids are not given to others.
        self._kept = (signature, lists, [type(None) if m is None else ref(m) for m in momenta],
                      [p for group in self.param_groups for p in group["params"]], list(self.state))
        return lists

    def _prepare_group(self, gi: int, group) -> list:
        """Checks every (param, grad, exp_avg) triple of the group, creates missing momentum, and
        returns one prepared launch (a `_TensorList`) per (device, dtype, momentum dtype)."""
        buckets: Dict[tuple, Tuple[List[Tensor], List[Tensor], List[Tensor]]] = {}
        for param in group["params"]:
            grad = param.grad
            if grad is None:
                continue
            state = self.state[param]
            if "exp_avg" not in state:
                state["exp_avg"] = torch.zeros_like(
                    param, dtype=self._momentum_dtype or param.dtype, memory_format=torch.preserve_format)
            exp_avg = state["exp_avg"]
            _check_triple(param, grad, exp_avg)
            key = (gi, param.device.index, param.dtype, exp_avg.dtype)
            ps, gs, ms = buckets.setdefault(key, ([], [], []))
            ps.append(param)
            gs.append(grad)
            ms.append(exp_avg)
        return [_TensorList(key, ps, gs, ms) for key, (ps, gs, ms) in buckets.items()]

    @torch.no_grad()
    def step(self) -> None:
        """Parameter and momentum update (no closure, no return value: lion_optimizer.py:57)."""
        self.grad_norm = None
        if self._zero is not None:
            self._zero.step()
            return
        lib = _lib.load()
        prepared = self._prepared()
        clip = None
        if self.max_grad_norm is not None:
            clip = self._clip_factor(prepared)
            if clip is None:
                return  # no parameter has a gradient
        for group, lists in zip(self.param_groups, prepared):
            lr = float(group["lr"])
            weight_decay = float(group["weight_decay"])
            beta1, beta2 = (float(b) for b in group["betas"])
            for tl in lists:
                args = (tl.params, tl.grads, tl.moms, tl.numels, tl.n, tl.p_code, tl.p_code, tl.m_code,
                        lr, beta1, beta2, weight_decay)
                where = (tl.device_index, _lib.current_stream_ptr(tl.device_index))
                if clip is None:
                    _lib.check(lib.fo_lion_multi_tensor_step(*args, *where))
                else:
                    _lib.check(lib.fo_lion_multi_tensor_step_clipped(*args, clip.data_ptr(), *where))

    def _clip_factor(self, prepared: List[list]) -> Optional[Tensor]:
        """Launches the norm over the gradients of all groups; returns a device buffer whose first float
        is the clipping factor, or None when no parameter has a gradient."""
        max_norm = self._checked_max_norm()
        lists = [tl for group_lists in prepared for tl in group_lists]
        if self._grad_list is None or len(self._grad_list[0]) != len(lists) or not all(map(is_, self._grad_list[0], lists)):
            grads = [p.grad for group in self.param_groups for p in group["params"] if p.grad is not None]
            self._grad_list = (lists, GradList(grads) if grads else None)
        if self._grad_list[1] is None:
            return None
        self.grad_norm, buffer = self._grad_list[1].launch(max_norm)
        return buffer

    def _checked_max_norm(self) -> float:
        max_norm = float(self.max_grad_norm)
        if not max_norm > 0:
            raise RuntimeError(f"max_grad_norm must be positive, got {max_norm}")
        return max_norm

    def load_state_dict(self, state_dict) -> None:
        """As torch.optim.Optimizer.load_state_dict; in process_group mode the loaded momentum
        (this rank's slices, as state_dict() saved them) is copied back into the rank's shard."""
        super().load_state_dict(state_dict)
        self._kept = self._grad_list = None  # the momentum tensors are new objects
        if self._zero is not None:
            self._zero.adopt_loaded_state()

    # -- ZeRO-1 accessors ------------------------------------------------------------------
    @property
    def flat_params(self) -> Optional[Tensor]:
        return None if self._zero is None else self._zero.flat_p

    @property
    def flat_grads(self) -> Optional[Tensor]:
        return None if self._zero is None else self._zero.flat_g


class _Zero1State:
    """Flat parameter / gradient buffers, this rank's momentum shard and the step that uses them.

    Every parameter becomes a view into `flat_p`; `p.grad` is pre-set to a view into `flat_g`
    so that backward accumulates straight into it (a caller that assigns other gradient
    tensors pays one copy per tensor in step()).  Gradient averaging across ranks is the
    caller's job (reduce-scatter or all-reduce before step()); the optimizer's one collective is
    the all-gather of updated weights.
    """

    def __init__(self, opt: Lion, group, momentum_dtype: Optional[torch.dtype], fused_gather: bool = False,
                 reduce_gradients: bool = False):
        import torch.distributed as dist

        self.reduce_gradients = reduce_gradients
        self.opt = opt
        self.group = group
        self.world = dist.get_world_size(group)
        self.rank = dist.get_rank(group)
        params = [p for g in opt.param_groups for p in g["params"]]
        if not params:
            raise RuntimeError("no parameters")
        if len(opt.param_groups) != 1:
            raise RuntimeError("process_group mode supports a single param group")
        dtype, device = params[0].dtype, params[0].device
        for p in params:
            if p.dtype != dtype or p.device != device:
                raise RuntimeError("process_group mode needs all parameters on one device with one dtype")
        self.params = params
        self.layout = FlatLayout.build([p.numel() for p in params], self.world)
        self.symm = None
        self.peer_ptrs: List[int] = []
        if fused_gather and self.world > 1:
            # peer-mapped allocation: every rank can store into every other rank's buffer
            import torch.distributed._symmetric_memory as symm_mem

            self.flat_p = symm_mem.empty(self.layout.total, dtype=dtype, device=device)
            self.flat_p.zero_()
            self.symm = symm_mem.rendezvous(self.flat_p, group)
            ptrs = list(self.symm.buffer_ptrs)
            self.peer_ptrs = [int(ptrs[r]) for r in range(self.world) if r != self.rank]
        else:
            self.flat_p = torch.zeros(self.layout.total, dtype=dtype, device=device)
        self.flat_g = torch.zeros(self.layout.total, dtype=dtype, device=device)
        self._grad_views: List[Tensor] = []
        with torch.no_grad():
            for p, off in zip(params, self.layout.offsets):
                n = p.numel()
                view = self.flat_p[off:off + n].view(p.shape)
                view.copy_(p.data.contiguous())
                p.data = view
                gview = self.flat_g[off:off + n].view(p.shape)
                if p.grad is not None:
                    gview.copy_(p.grad)
                p.grad = gview
                self._grad_views.append(gview)
        self.begin, self.end = self.layout.shard_range(self.rank)
        self.m_shard = torch.zeros(self.end - self.begin, dtype=momentum_dtype or dtype, device=device)
        for i, p in enumerate(params):
            _, s0, n = self.layout.tensor_slice_in_shard(i, self.rank)
            opt.state[p]["exp_avg"] = self.m_shard[s0:s0 + n]
        self.flat_step_fn = _flat_step
        # the two halves of the clipping factor, around the all-reduce of the sum of squares
        self.sumsq_fn, self.finish_norm_fn = shard_sumsq, finish_norm

    def adopt_loaded_state(self) -> None:
        """After Optimizer.load_state_dict: state[p]["exp_avg"] holds fresh tensors; copy them
        into the shard and point the state back at views of it."""
        with torch.no_grad():
            for i, p in enumerate(self.params):
                _, s0, n = self.layout.tensor_slice_in_shard(i, self.rank)
                view = self.m_shard[s0:s0 + n]
                loaded = self.opt.state[p].get("exp_avg")
                if loaded is not None and loaded.data_ptr() != view.data_ptr():
                    if loaded.numel() != n:
                        raise RuntimeError("loaded exp_avg does not match this rank's slice of the parameter")
                    view.copy_(loaded.reshape(-1))
                self.opt.state[p]["exp_avg"] = view

    def _average_gradients(self) -> None:
        import torch.distributed as dist

        shard = self.flat_g[self.begin:self.end]
        if dist.get_backend(self.group) == "gloo":  # no reduce-scatter there: all-reduce, keep the slice
            dist.all_reduce(self.flat_g, group=self.group)
            shard.div_(self.world)
        else:
            dist.reduce_scatter_tensor(shard, self.flat_g, op=dist.ReduceOp.AVG, group=self.group)

    def _clip_factor(self) -> Tensor:
        """Sum of squares of this rank's slice, added up over the ranks (every element of the flat
        gradient lies in one slice), then the factor: the same on all ranks."""
        import torch.distributed as dist

        max_norm = self.opt._checked_max_norm()
        sumsq = self.sumsq_fn(self.flat_g, self.begin, self.end)
        if self.world > 1:
            dist.all_reduce(sumsq, group=self.group)
        self.opt.grad_norm, coef = self.finish_norm_fn(sumsq, max_norm)
        return coef

    @torch.no_grad()
    def step(self) -> None:
        import torch.distributed as dist

        for p, gview in zip(self.params, self._grad_views):
            if p.grad is None:
                raise RuntimeError("process_group mode needs a gradient for every parameter")
            if p.grad.data_ptr() != gview.data_ptr():
                gview.copy_(p.grad)
                p.grad = gview
        if self.reduce_gradients and self.world > 1:
            self._average_gradients()
        group = self.opt.param_groups[0]
        clip = {} if self.opt.max_grad_norm is None else {"clip": self._clip_factor()}
        if self.symm is not None:
            # ranks meet before any of them overwrites a peer's weights, and again before any of
            # them reads the gathered result (device-side barriers on the current stream)
            self.symm.barrier(channel=0)
            _flat_step_push(self.flat_p, self.flat_g, self.m_shard, self.begin, self.end, self.peer_ptrs,
                            group["lr"], group["betas"], group["weight_decay"], **clip)
            self.symm.barrier(channel=1)
            return
        self.flat_step_fn(self.flat_p, self.flat_g, self.m_shard, self.begin, self.end, group["lr"],
                          group["betas"], group["weight_decay"], **clip)
        if self.world > 1:
            dist.all_gather_into_tensor(self.flat_p, self.flat_p[self.begin:self.end], group=self.group)
