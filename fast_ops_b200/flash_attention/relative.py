"""Attention with a learned relative position bias, differentiable in the bias.

The bias of query i and key j is table[bucket(j - (i + query_offset)), head]: near positions have a
bucket each, far ones share buckets that grow with the distance.  It is never materialised: the
kernels read it as one vector per head, add a constant away from the diagonal, and sum the table's
gradient where the backward forms dS.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib
from .flash_attention import _CODES, _I64x3, _prepare_bias, next_dropout_rng, recorded

_I64x2 = ctypes.c_int64 * 2
#: buckets of one side (the C ABI passes their starts in kernel arguments)
MAX_BUCKETS_PER_SIDE = 256


@lru_cache(maxsize=1024)
def _strides(strides: Tuple[int, ...]):
    """(batch, head, row) strides of a (B, H, S, D) tensor for the C ABI, which only reads them: a model's
    calls have few different ones."""
    return _I64x3(*strides[:3])


@lru_cache(maxsize=1024)
def _table_strides(strides: Tuple[int, int]):
    return _I64x2(*strides)


@lru_cache(maxsize=64)
def relative_bucket_starts(num_buckets: int, max_distance: int, bidirectional: bool) -> Tuple[int, ...]:
    """The smallest distance of each bucket of one side.

    With h buckets on a side (half of `num_buckets` if bidirectional, otherwise all) and e = h // 2,
    distances below e have a bucket each; bucket e + x starts at the smallest n with
    (n / e)^(h - e) >= (max_distance / e)^x: equal steps of the logarithm, up to `max_distance`, decided
    in whole numbers.  The last bucket takes everything beyond.  Positions after the query come
    second, from bucket h on; one-sided, they all count as distance 0.
    """
    if num_buckets < 2 or (bidirectional and (num_buckets < 4 or num_buckets % 2)):
        raise RuntimeError(f"num_buckets must be at least 2, or even and at least 4 if bidirectional, got {num_buckets}")
    per_side = num_buckets // 2 if bidirectional else num_buckets
    if per_side > MAX_BUCKETS_PER_SIDE:
        raise RuntimeError(f"at most {MAX_BUCKETS_PER_SIDE} buckets per side, got {per_side}")
    exact = per_side // 2
    if not exact < max_distance < 2**29:
        raise RuntimeError(f"max_distance must be above {exact} and below 2^29, got {max_distance}")
    steps = per_side - exact
    starts = list(range(exact))
    for x in range(steps):
        bound = max_distance**x * exact ** (steps - x)  # n^steps >= bound
        n = max(starts[-1] if starts else 0, int(math.exp(math.log(max_distance / exact) * x / steps) * exact) - 2, exact)
        while n**steps < bound:
            n += 1
        while n > exact and (n - 1) ** steps >= bound:
            n -= 1
        starts.append(n)
    return tuple(starts)


@lru_cache(maxsize=64)
def _starts_array(num_buckets: int, max_distance: int, bidirectional: bool):
    starts = relative_bucket_starts(num_buckets, max_distance, bidirectional)
    return (ctypes.c_int * len(starts))(*starts), len(starts)


@lru_cache(maxsize=256)
def _workspace_bytes(H: int, M: int, N: int, num_buckets: int, max_distance: int, bidirectional: bool, offset: int,
                     bias_rows: int) -> int:
    starts, n = _starts_array(num_buckets, max_distance, bidirectional)
    size = _lib.load().fo_rel_attn_workspace(H, M, N, starts, n, int(bidirectional), offset, bias_rows)
    _lib.check(-1 if size < 0 else 0)
    return size


@lru_cache(maxsize=256)
def _partial_floats(B: int, H: int, M: int, N: int, D: int, num_buckets: int, dropout: bool) -> int:
    size = _lib.load().fo_rel_attn_bwd_workspace(B, H, M, N, D, num_buckets, int(dropout))
    _lib.check(-1 if size < 0 else 0)
    return size // 4


class _Call:
    """The checked arguments of one call, shared by forward and backward."""

    def __init__(self, Q: Tensor, K: Tensor, V: Tensor, table: Tensor, max_distance: int, bidirectional: bool,
                 query_offset: int, causal: bool, softmax_scale: Optional[float], dropout_p: float,
                 rng: Optional[Tuple[int, int]]):
        if not (isinstance(Q, Tensor) and isinstance(K, Tensor) and isinstance(V, Tensor) and isinstance(table, Tensor)):
            raise RuntimeError("Q, K, V and table must be tensors")
        q_shape, k_shape, table_shape = Q.shape, K.shape, table.shape
        if len(q_shape) != 4 or len(k_shape) != 4:
            raise RuntimeError("Q, K, V must be 4-D")
        index = Q.get_device()
        if index < 0:
            raise RuntimeError("fast_ops_b200 attention needs CUDA tensors (there is no CPU path)")
        if K.get_device() != index or V.get_device() != index or table.get_device() != index:
            raise RuntimeError("Q, K, V and table must be on the same device")
        dtype = Q.dtype
        code = _CODES.get(dtype)
        if code is None:
            raise RuntimeError(f"inputs must be float16 or bfloat16, got {dtype}")
        if K.dtype != dtype or V.dtype != dtype:
            raise RuntimeError("Q, K, V must have the same dtype")
        table_code = code if table.dtype == dtype else _lib.FO_F32
        if table_code != code and table.dtype != torch.float32:
            raise RuntimeError(f"table must be float32 or have Q's dtype, got {table.dtype}")
        B, H, M, D = q_shape
        if k_shape[0] != B or k_shape[1] != H or k_shape[3] != D or V.shape != k_shape:
            raise RuntimeError(f"shape mismatch: Q {tuple(q_shape)}, K {tuple(k_shape)}, V {tuple(V.shape)}")
        if len(table_shape) != 2 or table_shape[1] != H:
            raise RuntimeError(f"table must be (num_buckets, {H}), got {tuple(table_shape)}")
        if D > 128 or D % 8 != 0 or D == 0:
            raise RuntimeError(f"head_dim must be a multiple of 8 and <= 128, got {D}")
        if Q.stride(3) != 1 or K.stride(3) != 1 or V.stride(3) != 1:
            raise RuntimeError("Q, K, V: the last dimension must be contiguous")
        if not 0.0 <= dropout_p < 1.0:
            raise RuntimeError(f"dropout_p must be in [0, 1), got {dropout_p}")
        if not 0 <= query_offset <= 2**29:
            raise RuntimeError(f"query_offset must be in [0, 2^29], got {query_offset}")
        self.B, self.H, self.M, self.D, self.N = B, H, M, D, k_shape[2]
        self.code, self.device, self.index, self.table_code = code, Q.device, index, table_code
        self.num_buckets = table_shape[0]
        self.key = key = (self.num_buckets, int(max_distance), bool(bidirectional))
        self.starts, self.n_starts = _starts_array(*key)
        self.bidirectional, self.offset, self.causal = int(key[2]), int(query_offset), 1 if causal else 0
        self.scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
        self.dropout_p = float(dropout_p)
        if rng is not None:
            rng = (rng[0] & (2**64 - 1), rng[1] & (2**64 - 1))
        elif self.dropout_p > 0.0:
            rng = next_dropout_rng(Q.device, B * H * M * self.N)
        self.rng = rng or (0, 0)

    def bias(self, bias: Optional[Tensor], Q: Tensor):
        if bias is None:
            return None, 0, (None, None, _lib.FO_F32)
        if bias.dim() == 4 and bias.shape[2] != 1:
            raise RuntimeError("beside a relative bias, bias must be (1 or B, 1 or H, 1, N): the same for every query")
        kept, ptr, strides, code = _prepare_bias(bias, Q, self.B, self.H, self.M, self.N)
        strides[2] = 0  # a single query row's stride says nothing
        rows = (self.B if strides[0] else 1) * (self.H if strides[1] else 1)
        return kept, rows, (ptr, strides, code)

    def forward(self, Q: Tensor, K: Tensor, V: Tensor, table: Tensor, bias: Optional[Tensor], lse: bool):
        """(O, LSE or None, the expanded bias or None where nothing reads it)."""
        O = torch.empty_like(Q, memory_format=torch.contiguous_format)
        lse_t = Q.new_empty((self.B, self.H, self.M), dtype=torch.float32) if lse else None
        # Kept for the backward, which takes from the strides where in the workspace the rows of the bias lie; the saved
        # tensors may come back with other strides than they left with (saved_tensors_hooks, save_on_cpu).
        self.kept_bias, rows, self.bias_args = self.bias(bias, Q)
        workspace = None
        if lse or self.M > 1 or self.dropout_p > 0.0:
            workspace = torch.empty(_workspace_bytes(self.H, self.M, self.N, *self.key, self.offset, rows),
                                    dtype=torch.uint8, device=self.device)
        _lib.check(_lib.load().fo_rel_attn_fwd(
            Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), lse_t.data_ptr() if lse else None,
            self.B, self.H, self.M, self.N, self.D,
            _strides(Q.stride()), _strides(K.stride()), _strides(V.stride()), _strides(O.stride()),
            self.code, self.causal, self.scale, table.data_ptr(), _table_strides(table.stride()), self.table_code,
            self.starts, self.n_starts, self.bidirectional, self.offset,
            None if workspace is None else workspace.data_ptr(), *self.bias_args, self.dropout_p, *self.rng, self.index,
            _lib.current_stream_ptr(self.index)))
        return O, lse_t, workspace

    def backward(self, dO: Tensor, Q: Tensor, K: Tensor, V: Tensor, O: Tensor, LSE: Tensor, workspace: Tensor,
                 table_grad: Optional[torch.dtype]):
        """(dQ, dK, dV, the table's gradient or None), after `forward`."""
        sb, sh, ss, sd = dO.stride()
        if sd != 1 or sb % 8 or sh % 8 or ss % 8 or not (sb and sh and ss) or dO.data_ptr() % 16:
            # broadcast or cut from a larger tensor (where it may be dense and still begin between two 16-byte addresses)
            dO = dO.clone(memory_format=torch.contiguous_format)
        if K.stride(1) == 0 or V.stride(1) == 0:
            # one K/V head for all query heads: one dK, dV per query head needs storage of its own
            # (autograd sums them through the expand)
            K, V = K.contiguous(), V.contiguous()
        dQ, dK, dV = torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)
        for t in (dQ, dK, dV):
            if t.stride(3) != 1:
                raise RuntimeError("gradient layout: the last dimension must be contiguous")
        lib = _lib.load()
        rows = self.B * self.H * self.M
        partials = 0
        dtable = None
        if table_grad is not None:
            dtable = torch.empty((self.num_buckets, self.H), dtype=table_grad, device=self.device)
            partials = _partial_floats(self.B, self.H, self.M, self.N, self.D, self.num_buckets, self.dropout_p > 0.0)
        # one scratch block: the fp32 dQ accumulator (B, H, M, D), the table's partial sums, rowsum(O o dO) (B, H, M)
        scratch = torch.empty(rows * (self.D + 1) + partials, dtype=torch.float32, device=self.device)
        dq_accum = scratch.data_ptr()
        partial_sums = dq_accum + 4 * rows * self.D  # a multiple of 32 bytes on, since D is one of 8
        _lib.check(lib.fo_rel_attn_bwd(
            Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), dO.data_ptr(), LSE.data_ptr(), dQ.data_ptr(),
            dK.data_ptr(), dV.data_ptr(), None if dtable is None else dtable.data_ptr(), dq_accum,
            partial_sums + 4 * partials, partial_sums,
            self.B, self.H, self.M, self.N, self.D,
            _strides(Q.stride()), _strides(K.stride()), _strides(V.stride()), _strides(O.stride()), _strides(dO.stride()),
            _strides(dQ.stride()), _strides(dK.stride()), _strides(dV.stride()), self.code, self.causal,
            self.scale, self.table_code, self.starts, self.n_starts, self.bidirectional, self.offset,
            workspace.data_ptr(), *self.bias_args, self.dropout_p, *self.rng, self.index,
            _lib.current_stream_ptr(self.index)))
        return dQ, dK, dV, dtable


class _RelativeAttentionFunction(Function):
    @staticmethod
    def forward(ctx, Q: Tensor, K: Tensor, V: Tensor, table: Tensor, call: _Call, bias: Optional[Tensor],
                return_lse: bool):
        O, lse, workspace = call.forward(Q, K, V, table, bias, True)
        ctx.save_for_backward(Q, K, V, O, lse, workspace)
        ctx.call, ctx.table_dtype = call, table.dtype
        if not return_lse:
            return O
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(lse)
        return O, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dO: Optional[Tensor], _dlse=None):
        if dO is None:
            return (None,) * 7
        Q, K, V, O, lse, workspace = ctx.saved_tensors
        return ctx.call.backward(dO, Q, K, V, O, lse, workspace,
                                 ctx.table_dtype if ctx.needs_input_grad[3] else None) + (None,) * 3


def relative_attention(Q: Tensor, K: Tensor, V: Tensor, table: Tensor, *, max_distance: int = 128,
                       bidirectional: bool = True, query_offset: int = 0, causal: bool = False,
                       softmax_scale: Optional[float] = None, return_lse: bool = False,
                       bias: Optional[Tensor] = None, dropout_p: float = 0.0,
                       rng: Optional[Tuple[int, int]] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """softmax(scale * Q K^T + table[bucket(j - i - query_offset)] [+ bias] [+ causal mask]) V.

    Q: (B, H, M, D); K, V: (B, H, N, D); fp16 or bf16, layouts as in `multi_head_attention` (K and V may
    be expanded over the heads).  Differentiable in Q, K, V and `table`, once and in reverse mode.

    :param table: (num_buckets, H), fp32 or Q's dtype, any non-negative strides; entries of -1e6 and below
        mask the keys of their bucket, as -inf does.
    :param max_distance, bidirectional: the buckets, see `relative_bucket_starts`.  Bidirectional, keys
        before and after the query have num_buckets / 2 buckets each; otherwise all buckets are for the
        keys before it and those after it are at distance 0 (as a causal model wants it).
    :param query_offset: key position of query row 0.  A decoder that has N keys stored and asks for the
        last M of them passes N - M; a single query row runs in the decoding kernel.
    :param causal: masks keys j > i + query_offset.
    :param bias: added beside the learned bias, not differentiable: (1 or B, 1 or H, 1, N), fp32 or Q's
        dtype; entries of -1e6 and below mask keys (padding), as -inf does.  A query row whose keys are
        all masked gives zeros, and no gradients.
    :param dropout_p, rng: as in `flash_attention_forward`; without `rng` the mask is drawn from the
        device's default generator, as in `multi_head_attention`.
    :returns: O (B, H, M, D), contiguous, or (O, LSE) with `return_lse`.

    Violations of these raise RuntimeError.  The table's gradient is summed in an order that does not
    change from run to run.  P and dS are rounded to Q's dtype for their matmuls, as in the framework's other
    attention calls; everything else is fp32 or wider.  While a backward runs it holds scratch for the
    table's gradient that grows with M N: 4 to 8 bytes for every 32 x 32 scores (fo_rel_attn_bwd_workspace).
    """
    call = _Call(Q, K, V, table, max_distance, bidirectional, query_offset, causal, softmax_scale, dropout_p, rng)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("the gradient of bias is not supported (that of table is)")
    if recorded(Q, K, V, table):
        return _RelativeAttentionFunction.apply(Q, K, V, table, call, bias, return_lse)
    O, lse, _ = call.forward(Q, K, V, table, bias, return_lse)
    return (O, lse) if return_lse else O
