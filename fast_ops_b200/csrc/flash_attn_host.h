// Host functions of the attention calls that more than one translation unit uses.
#pragma once

#include <cuda.h>

#include "flash_attn_bwd.cuh"
#include "flash_attn_common.cuh"

namespace fo {

// Validates the optional bias / dropout arguments of the extended entry points and fills `ex` (flash_attn_fwd.cu).
int make_attn_extras(AttnExtras* ex, const void* bias, const int64_t* bias_strides, int bias_dtype, int dtype,
                     float dropout_p, uint64_t rng_seed, uint64_t rng_offset);

// A relative position bias as the entry points get it.
struct RelArgs {
  RelBuckets buckets;
  const void* table;
  int64_t stride_bucket, stride_head;  // elements
  int table_f32;                       // 1: fp32, 0: the 16-bit type of q
  RelBias bias;                        // what the tile kernels read
  void* dtable;                        // backward: the table's gradient, of table_dtype, or null
  int table_dtype;
  int64_t bias_rows;                   // rows of the expanded vector bias, of bias_heads heads each
  int bias_heads;
};

// The forward and the backward behind all entry points (flash_attn_fwd.cu, flash_attn_bwd.cu).
int attn_fwd_impl(const void* q, const void* k, const void* v, void* o, float* lse,
                  int B, int H, int Sq, int Sk, int D,
                  const int64_t q_strides[3], const int64_t k_strides[3],
                  const int64_t v_strides[3], const int64_t o_strides[3],
                  int dtype, int causal, float softmax_scale, const AttnExtras* ex, const RelArgs* rel,
                  int device, void* stream);
int attn_bwd_impl(const void* q, const void* k, const void* v, const void* o, const void* dout,
                  const float* lse, void* dq, void* dk, void* dv, float* dq_accum, float* delta,
                  int B, int H, int Sq, int Sk, int D,
                  const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                  const int64_t o_strides[3], const int64_t do_strides[3],
                  const int64_t dq_strides[3], const int64_t dk_strides[3], const int64_t dv_strides[3],
                  int dtype, int causal, float softmax_scale, const AttnExtras* ex, const RelArgs* rel,
                  int device, void* stream);

// The launches of the kernels built for a relative bias (flash_attn_rel.cu), called by the two above.
// The bias is brought into the form they read by launch_rel_expand before the first of them.  `half_tiles`:
// tk and tv have boxes of 64 keys, for the kernel with one query tile per CTA.
int launch_fwd_rel(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnParams& prm, bool half_tiles,
                   bool bf16, cudaStream_t stream);
int launch_bwd_rel(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                   const CUtensorMap& tdq, const AttnBwdParams& prm, bool bf16, cudaStream_t stream);
int launch_rel_expand(const RelArgs& rel, const AttnExtras& ex, int H, int Sk, float softmax_scale, bool bf16,
                      cudaStream_t stream);

// The table's gradient from the partial sums of launch_bwd_rel's kernel.
int launch_table_grad(const RelArgs& rel, int B, int H, int Sq, int Sk, int D, int causal, float softmax_scale, bool dropout,
                      cudaStream_t stream);

struct DecodeParams;
int launch_decode_rel(const DecodeParams& prm, const RelArgs& rel, const AttnExtras& ex, int B, int H, int Sk, int D,
                      bool shared_kv, bool bf16, int num_sms, int device, cudaStream_t stream);

}  // namespace fo
