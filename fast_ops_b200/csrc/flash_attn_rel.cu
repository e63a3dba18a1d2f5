// Attention with a learned relative position bias (rel_bias.cuh): entry points, the launches of the tile
// and decoding kernels built for it, and the two small kernels around them: the bias of a head as a vector
// over the relative position, and the gradient of the table from the backward's partial sums.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "flash_attn_bwd.cuh"
#include "flash_attn_decode.cuh"
#include "flash_attn_host.h"
#include "flash_attn_ws64r.cuh"
#include "flash_attn_ws64s.cuh"
#include "fo_host.h"

namespace {

using fo::RelArgs;
using fo::RelBias;
using fo::RelBuckets;

// The bias in the form the tile kernels read: values[h][s][x] = table[bucket(x + s - zero)][h] / scale, the
// buckets themselves, and the rows of a vector bias.  The first blocks make the former, 256 positions of one
// head each; then one block takes each row.
struct ExpandParams {
  RelBuckets buckets;
  const uint8_t* table;
  int64_t stride_bucket, stride_head;
  int table_f32;
  const uint8_t* bias;  // vector bias as the caller gave it, or null
  int64_t bias_stride_b, bias_stride_h;
  int bias_f32;
  int bias_heads;       // heads of the rows made of it
  float inv_scale;      // 1 / softmax scale
  int Sk, zero, width, stride, value_blocks, vec_width;
  float* values;
  int* bucket_of;
  float* vec;
  int4* vec_extent;
};

template <bool kBf16>
__global__ void __launch_bounds__(256)
rel_expand_kernel(const __grid_constant__ ExpandParams prm) {
  fo::grid_allow_next();
  const int per_head = (prm.width + 255) / 256;
  if (static_cast<int>(blockIdx.x) < prm.value_blocks) {
    const int h = blockIdx.x / per_head;
    const int x = (blockIdx.x - h * per_head) * 256 + threadIdx.x;
    if (x >= prm.width) return;
    const int bucket = fo::rel_bucket(prm.buckets, x - prm.zero);
    const float v = fo::scaled_or_masked(
        fo::load_elem<kBf16>(prm.table, bucket * prm.stride_bucket + h * prm.stride_head, prm.table_f32), prm.inv_scale);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (x >= s) prm.values[(static_cast<int64_t>(h) * 4 + s) * prm.stride + x - s] = v;
    if (h == 0) prm.bucket_of[x] = bucket;
    return;
  }
  const int row = blockIdx.x - prm.value_blocks;
  const int b = row / prm.bias_heads, h = row - b * prm.bias_heads;
  const int64_t src = b * prm.bias_stride_b + h * prm.bias_stride_h;
  float* const dst = prm.vec + static_cast<int64_t>(row) * prm.vec_width;
  int end = 0, first = prm.vec_width, last = -1;
#pragma unroll 4
  for (int key = threadIdx.x; key < prm.vec_width; key += 256) {
    const float v = key < prm.Sk ? fo::scaled_or_masked(fo::load_elem<kBf16>(prm.bias, src + key, prm.bias_f32), prm.inv_scale) : 0.f;
    dst[key] = v;
    if (v != 0.f) {
      first = min(first, key);
      last = key;
    }
    if (key < prm.Sk && !(v == __int_as_float(0xff800000))) end = key + 1;
  }
  first = __reduce_min_sync(0xffffffffu, first);
  last = __reduce_max_sync(0xffffffffu, last);
  end = __reduce_max_sync(0xffffffffu, end);
  __shared__ int found[8][3];
  if ((threadIdx.x & 31) == 0) {
    found[threadIdx.x >> 5][0] = first;
    found[threadIdx.x >> 5][1] = last;
    found[threadIdx.x >> 5][2] = end;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 8; ++w) {
    first = min(first, found[w][0]);
    last = max(last, found[w][1]);
    end = max(end, found[w][2]);
  }
  prm.vec_extent[row] = make_int4(end, first / 64, last < 0 ? 0 : last / 64 + 1, 0);
}

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The table's gradient from the backward's partial sums (which carry the softmax scale, as dS of the other
// gradients does): dtable[u][h] = 1 / scale * (sums of the parts that are far from the diagonal on the side
// of u's bucket + sums by bucket of the parts near it).
//
// dS = P o (dP - delta) sums to zero over the keys of a query.  delta comes from an O whose P and whose
// result were rounded to 16 bits; an error of it leaves P times that error in every dS of the row, with one
// sign, which the far buckets collect over thousands of keys: 0.5 to 1 % of their gradient at S = 4096 to 8192.
// What the sums over all keys of a block of queries miss zero by is that error's sum over the block; it
// is put back in proportion to the probability mass that each side holds of the block's queries.
// A cluster of kGradCtas blocks per head, whose partial results the first one adds up: a warp per (batch, block of
// queries) for the far sums, and rows of neighbouring buckets for the sums by bucket.  Everything in a fixed order
// and in double.  Bound by latency (the sums are a few MB at most): one block per head took 22 us at B16 H12 S512 and
// 18 at B2 H16 S4096, the cluster 9 and 14, most of which the rounding of dQ hides.
constexpr int kGradCtas = 8, kGradWarps = 8;

template <class T>
__global__ void __cluster_dims__(kGradCtas, 1, 1) __launch_bounds__(kGradWarps * 32)
rel_table_grad_kernel(const RelBias rel, T* __restrict__ dtable, int B, int H, int n_q_tiles, int n_k_tiles, int warps,
                      int causal, float inv_scale) {
  namespace cg = cooperative_groups;
  fo::grid_allow_next();  // the rounding of dQ, which does not depend on this
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double far[kGradWarps][2];
  __shared__ double cta_far[2];
  __shared__ double part[kGradWarps][32];
  __shared__ double cta_part[2 * fo::kRelMaxStarts];  // sum by bucket of this block's rows
  const int h = blockIdx.y;
  const int rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = warps / 4, cols = fo::kBlockM / parts;  // four warps share a part's queries
  double left = 0, right = 0;
  const uint32_t items = static_cast<uint32_t>(B) * n_q_tiles * parts;
  for (uint32_t item = rank * kGradWarps + warp; item < items; item += kGradCtas * kGradWarps) {
    const int p = static_cast<int>(item % parts);
    const uint32_t bi = item / parts;
    const int b = static_cast<int>(bi / n_q_tiles), i = static_cast<int>(bi - static_cast<uint32_t>(b) * n_q_tiles);
    const float2* const row = rel.tile_sums + ((static_cast<int64_t>(b) * H + h) * n_q_tiles + i) * n_k_tiles * warps + p * 4;
    const int q_first = i * fo::kBlockM + p * cols + rel.offset;  // key position of the part's first query
    // key tiles that this query tile sees and that have keys (the backward visits no others)
    int n = rel.vec == nullptr ? n_k_tiles : (fo::rel_keys(rel, b, h, n_k_tiles * fo::kBlockN) + fo::kBlockN - 1) / fo::kBlockN;
    if (causal) n = min(n, (i * fo::kBlockM + fo::kBlockM - 1 + rel.offset) / fo::kBlockN + 1);
    double ds = 0, mass = 0, ds_side[2] = {0, 0}, mass_side[2] = {0, 0};
#pragma unroll 4
    for (int x = lane; x < n * 4; x += 32) {
      const int key = x * 32;  // key tile x / 4, its quarter x % 4
      const float2 v = row[static_cast<int64_t>(x >> 2) * warps + (x & 3)];
      const int d_first = key - (q_first + cols - 1);
      const fo::RelSide side = fo::rel_side(rel, d_first, d_first + 30 + cols);
      ds += v.x;
      mass += v.y;
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (side == (w == 0 ? fo::kRelLeft : fo::kRelRight)) {
          ds_side[w] += v.x;
          mass_side[w] += v.y;
        }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      ds += __shfl_xor_sync(0xffffffffu, ds, off);
      mass += __shfl_xor_sync(0xffffffffu, mass, off);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        ds_side[w] += __shfl_xor_sync(0xffffffffu, ds_side[w], off);
        mass_side[w] += __shfl_xor_sync(0xffffffffu, mass_side[w], off);
      }
    }
    if (mass > 0) {
      left += ds_side[0] - ds * (mass_side[0] / mass);
      right += ds_side[1] - ds * (mass_side[1] / mass);
    }
  }
  if (lane == 0) {
    far[warp][0] = left;
    far[warp][1] = right;
  }
  // rows of the sums by bucket: (batch, key tile, warp), of which this block takes every kGradCtas-th
  const int per_batch = n_k_tiles * warps;
  const uint32_t rows = static_cast<uint32_t>(B) * per_batch;
  const int nb = rel.num_buckets;
  for (int u0 = 0; u0 < nb; u0 += 32) {
    const int u = u0 + lane;
    double sum = 0;
    if (u < nb) {
#pragma unroll 8
      for (uint32_t r = rank * kGradWarps + warp; r < rows; r += kGradCtas * kGradWarps) {
        const uint32_t b = r / per_batch;  // row (b * H + h) * per_batch + r - b * per_batch
        sum += static_cast<double>(rel.acc[(static_cast<int64_t>(b * (H - 1) + h) * per_batch + r) * nb + u]);
      }
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && u < nb) {
      for (int i = 1; i < kGradWarps; ++i) sum += part[i][lane];
      cta_part[u] = sum;
    }
    __syncthreads();
  }
  if (threadIdx.x < 2) {
    double sum = 0;
    for (int i = 0; i < kGradWarps; ++i) sum += far[i][threadIdx.x];
    cta_far[threadIdx.x] = sum;
  }
  cluster.sync();
  if (rank == 0) {
    const int left_bucket = rel.bucket_of[0], right_bucket = rel.bucket_of[rel.width - 1];
    for (int u = threadIdx.x; u < nb; u += kGradWarps * 32) {
      double sum = 0;
      for (int c = 0; c < kGradCtas; ++c) {
        sum += cluster.map_shared_rank(cta_part, c)[u];
        if (u == left_bucket) sum += cluster.map_shared_rank(cta_far, c)[0];
        if (u == right_bucket) sum += cluster.map_shared_rank(cta_far, c)[1];
      }
      dtable[static_cast<int64_t>(u) * H + h] = from_f32<T>(static_cast<float>(sum * inv_scale));
    }
  }
  cluster.sync();  // no block leaves while its shared memory is being read
}

// Checks of the buckets and of where the queries stand; fills everything of `rel` but the table and the device
// pointers of the expanded vector.
int make_rel_args(RelArgs* rel, int H, int Sq, int Sk, const int* starts, int n_starts, int two_sided, int query_offset) {
  FO_REQUIRE(starts, "null bucket starts");
  FO_REQUIRE(n_starts >= 1 && n_starts <= fo::kRelMaxStarts, "1 to %d buckets per side (got %d)", fo::kRelMaxStarts, n_starts);
  FO_REQUIRE(starts[0] == 0, "the first bucket must start at distance 0");
  for (int i = 1; i < n_starts; ++i) FO_REQUIRE(starts[i] >= starts[i - 1], "bucket starts must not descend");
  FO_REQUIRE(query_offset >= 0 && query_offset <= (1 << 29), "query_offset must be in [0, 2^29] (got %d)", query_offset);
  FO_REQUIRE(Sq > 0 && Sk > 0 && Sq <= (1 << 29) && Sk <= (1 << 29), "Sq and Sk must be in [1, 2^29]");
  std::memset(rel, 0, sizeof(*rel));
  std::copy(starts, starts + n_starts, rel->buckets.starts);
  rel->buckets.n = n_starts;
  rel->buckets.two_sided = two_sided ? 1 : 0;
  RelBias& bias = rel->bias;
  bias.offset = query_offset;
  bias.num_buckets = n_starts * (two_sided ? 2 : 1);
  // no relative position of the call lies beyond these
  const int last = starts[n_starts - 1];
  bias.far_left = std::min(last, Sq + query_offset);
  bias.far_right = two_sided ? std::min(std::max(last, 1), Sk) : 0;
  bias.zero = bias.far_left + fo::kRelMargin;
  bias.width = bias.zero + bias.far_right + fo::kRelMargin + 1;
  bias.stride = (bias.width - 8 + 31) / 32 * 32 + 8;
  FO_REQUIRE(H <= 0 || 4LL * H * bias.stride < (1LL << 31), "too many heads for bucket starts up to %d", last);
  return FO_OK;
}

// The type that the table or its gradient has.
int check_table_dtype(int table_dtype, int dtype) {
  FO_REQUIRE(dtype == FO_F16 || dtype == FO_BF16, "attention inputs must be fp16 or bf16 (got dtype %d)", dtype);
  FO_REQUIRE(table_dtype == FO_F32 || table_dtype == dtype, "the table must be fp32 or have the dtype of q (got dtype %d)",
             table_dtype);
  return FO_OK;
}

int set_table(RelArgs* rel, const void* table, int table_dtype, const int64_t* table_strides, int dtype) {
  FO_REQUIRE(table && table_strides, "null relative bias argument");
  if (int rc = check_table_dtype(table_dtype, dtype)) return rc;
  FO_REQUIRE(reinterpret_cast<uintptr_t>(table) % (table_dtype == FO_F32 ? 4 : 2) == 0, "the table is not aligned to its elements");
  FO_REQUIRE(table_strides[0] >= 0 && table_strides[1] >= 0, "the table's strides must be non-negative");
  rel->table = table;
  rel->stride_bucket = table_strides[0];
  rel->stride_head = table_strides[1];
  rel->table_f32 = table_dtype == FO_F32;
  return FO_OK;
}

// The expanded bias in a workspace: values, rows of the vector bias, buckets.
int64_t expanded_bytes(const RelBias& bias, int H, int64_t bias_rows, int Sk) {
  const int64_t width = fo::rel_vec_width(Sk);
  return (static_cast<int64_t>(H) * 4 * bias.stride + bias_rows * width + bias.stride) * 4 + bias_rows * 16;
}

int set_expanded(RelArgs* rel, void* workspace, const fo::AttnExtras& ex, int B, int H, int Sk, bool needed) {
  if (!needed) return FO_OK;
  FO_REQUIRE(workspace != nullptr, "null workspace");
  FO_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "workspace must be 16-byte aligned");
  FO_REQUIRE(B > 0 && H > 0, "B and H must be positive (got %d %d)", B, H);
  RelBias& bias = rel->bias;
  bias.values = static_cast<const float*>(workspace);
  const float* next = bias.values + static_cast<int64_t>(H) * 4 * bias.stride;
  if (ex.bias != nullptr) {
    // one row for each batch and head that has its own; where the caller's bias is broadcast, the row is too
    rel->bias_heads = ex.bias_stride_h != 0 ? H : 1;
    rel->bias_rows = static_cast<int64_t>(ex.bias_stride_b != 0 ? B : 1) * rel->bias_heads;
    bias.vec_width = fo::rel_vec_width(Sk);
    bias.vec = next;
    bias.vec_row_b = ex.bias_stride_b != 0 ? rel->bias_heads : 0;
    bias.vec_row_h = ex.bias_stride_h != 0 ? 1 : 0;
    next += rel->bias_rows * bias.vec_width;
  }
  bias.bucket_of = reinterpret_cast<const int*>(next);
  bias.vec_extent = reinterpret_cast<const int4*>(bias.bucket_of + bias.stride);  // every part is a multiple of 16 bytes
  return FO_OK;
}

// Warps of the backward that sum for the table's gradient, per key tile.
int bwd_warps(int D, bool dropout) {
  if (D > 64) return dropout ? fo::BwdConfig<128, fo::kBwdRelBias | fo::kBwdDropout>::kComputeWarps
                             : fo::BwdConfig<128, fo::kBwdRelBias>::kComputeWarps;
  return dropout ? fo::BwdConfig<64, fo::kBwdRelBias | fo::kBwdDropout>::kComputeWarps
                 : fo::BwdConfig<64, fo::kBwdRelBias>::kComputeWarps;
}

// Floats of the backward's partial sums: float2 per tile and warp first, then the sums by bucket.
int64_t tile_sum_floats(int B, int H, int Sq, int Sk, int D, bool dropout) {
  return 2LL * B * H * ((Sq + fo::kBlockM - 1) / fo::kBlockM) * ((Sk + fo::kBlockN - 1) / fo::kBlockN) * bwd_warps(D, dropout);
}

int64_t bucket_sum_floats(int B, int H, int Sk, int D, int num_buckets, bool dropout) {
  return 1LL * B * H * ((Sk + fo::kBlockN - 1) / fo::kBlockN) * bwd_warps(D, dropout) * num_buckets;
}

int check_bias_strides(const void* bias, const int64_t* strides) {
  if (bias == nullptr) return FO_OK;
  FO_REQUIRE(strides != nullptr, "bias given without strides");
  FO_REQUIRE(strides[2] == 0, "beside a relative bias, bias must be the same for every query row (row stride 0)");
  return FO_OK;
}

}  // namespace

namespace fo {

int launch_rel_expand(const RelArgs& rel, const AttnExtras& ex, int H, int Sk, float softmax_scale, bool bf16,
                      cudaStream_t stream) {
  ExpandParams prm;
  prm.buckets = rel.buckets;
  prm.table = static_cast<const uint8_t*>(rel.table);
  prm.stride_bucket = rel.stride_bucket;
  prm.stride_head = rel.stride_head;
  prm.table_f32 = rel.table_f32;
  prm.bias = static_cast<const uint8_t*>(ex.bias);
  prm.bias_stride_b = ex.bias_stride_b;
  prm.bias_stride_h = ex.bias_stride_h;
  prm.bias_f32 = ex.bias_f32;
  prm.bias_heads = rel.bias_heads;
  prm.inv_scale = 1.f / softmax_scale;
  prm.Sk = Sk;
  prm.zero = rel.bias.zero;
  prm.width = rel.bias.width;
  prm.stride = rel.bias.stride;
  prm.vec_width = rel_vec_width(Sk);
  prm.values = const_cast<float*>(rel.bias.values);
  prm.bucket_of = const_cast<int*>(rel.bias.bucket_of);
  prm.vec = const_cast<float*>(rel.bias.vec);
  prm.vec_extent = const_cast<int4*>(rel.bias.vec_extent);
  const int64_t value_blocks = static_cast<int64_t>((prm.width + 255) / 256) * H;
  const int64_t blocks = value_blocks + rel.bias_rows;
  FO_REQUIRE(blocks <= 0x7fffffff, "the bias is too large for one launch");
  prm.value_blocks = static_cast<int>(value_blocks);
  auto kernel = bf16 ? rel_expand_kernel<true> : rel_expand_kernel<false>;
  kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(prm);
  g_launch_count.fetch_add(1, std::memory_order_relaxed);
  FO_CUDA_CHECK(cudaGetLastError());
  return FO_OK;
}

int launch_fwd_rel(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const AttnParams& prm, bool half_tiles,
                   bool bf16, cudaStream_t stream) {
#define FO_REL_FORM(LAUNCH, DK, ...) \
  bf16 ? LAUNCH<DK, true, __VA_ARGS__>(tq, tk, tv, prm, stream) : LAUNCH<DK, false, __VA_ARGS__>(tq, tk, tv, prm, stream)
  const bool wide = prm.d_real > 64, vec = prm.rel.vec != nullptr;
  if (half_tiles) {
    if (wide && prm.d_real <= 96) return vec ? FO_REL_FORM(launch_ws64s, 128, 96, (kFwdRelBias | kFwdVecBias)) : FO_REL_FORM(launch_ws64s, 128, 96, kFwdRelBias);
    if (wide) return vec ? FO_REL_FORM(launch_ws64s, 128, 128, (kFwdRelBias | kFwdVecBias)) : FO_REL_FORM(launch_ws64s, 128, 128, kFwdRelBias);
    return vec ? FO_REL_FORM(launch_ws64s, 64, 64, (kFwdRelBias | kFwdVecBias)) : FO_REL_FORM(launch_ws64s, 64, 64, kFwdRelBias);
  }
  if (prm.ex.dropout) {
    if (wide) return vec ? FO_REL_FORM(launch_ws64r, 128, (kFwdRelBias | kFwdVecBias | kFwdDropout)) : FO_REL_FORM(launch_ws64r, 128, (kFwdRelBias | kFwdDropout));
    return vec ? FO_REL_FORM(launch_ws64r, 64, (kFwdRelBias | kFwdVecBias | kFwdDropout)) : FO_REL_FORM(launch_ws64r, 64, (kFwdRelBias | kFwdDropout));
  }
  if (wide) return vec ? FO_REL_FORM(launch_ws64r, 128, (kFwdRelBias | kFwdVecBias)) : FO_REL_FORM(launch_ws64r, 128, kFwdRelBias);
  return vec ? FO_REL_FORM(launch_ws64r, 64, (kFwdRelBias | kFwdVecBias)) : FO_REL_FORM(launch_ws64r, 64, kFwdRelBias);
#undef FO_REL_FORM
}

int launch_bwd_rel(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                   const CUtensorMap& tdq, const AttnBwdParams& prm, bool bf16, cudaStream_t stream) {
#define FO_REL_FORM(DK, ...) \
  bf16 ? launch_bwd<DK, true, __VA_ARGS__>(tq, tk, tv, tdo, tdq, prm, stream) : launch_bwd<DK, false, __VA_ARGS__>(tq, tk, tv, tdo, tdq, prm, stream)
  if (prm.d_real > 64) {
    if (prm.ex.dropout) return FO_REL_FORM(128, (kBwdRelBias | kBwdDropout));
    if (prm.d_real <= 96) return FO_REL_FORM(128, kBwdRelBias, 96);
    return FO_REL_FORM(128, kBwdRelBias);
  }
  if (prm.ex.dropout) return FO_REL_FORM(64, (kBwdRelBias | kBwdDropout));
  return FO_REL_FORM(64, kBwdRelBias);
#undef FO_REL_FORM
}

int launch_table_grad(const RelArgs& rel, int B, int H, int Sq, int Sk, int D, int causal, float softmax_scale, bool dropout,
                      cudaStream_t stream) {
  const int q_tiles = (Sq + kBlockM - 1) / kBlockM, k_tiles = (Sk + kBlockN - 1) / kBlockN;
  const int warps = bwd_warps(D, dropout);
  const float inv = 1.f / softmax_scale;
#define FO_TABLE_GRAD(T)                                                       \
  rel_table_grad_kernel<<<dim3(kGradCtas, H), kGradWarps * 32, 0, stream>>>(   \
      rel.bias, static_cast<T*>(rel.dtable), B, H, q_tiles, k_tiles, warps, causal ? 1 : 0, inv)
  if (rel.table_dtype == FO_F32) FO_TABLE_GRAD(float);
  else if (rel.table_dtype == FO_BF16) FO_TABLE_GRAD(__nv_bfloat16);
  else FO_TABLE_GRAD(__half);
#undef FO_TABLE_GRAD
  g_launch_count.fetch_add(1, std::memory_order_relaxed);
  FO_CUDA_CHECK(cudaGetLastError());
  return FO_OK;
}

int launch_decode_rel(const DecodeParams& prm, const RelArgs& args, const AttnExtras& ex, int B, int H, int Sk, int D,
                      bool shared_kv, bool bf16, int num_sms, int device, cudaStream_t stream) {
  DecodeRel rel;
  rel.buckets = args.buckets;
  rel.table = static_cast<const uint8_t*>(args.table);
  rel.stride_bucket = args.stride_bucket;
  rel.stride_head = args.stride_head;
  rel.table_f32 = args.table_f32;
  rel.offset = args.bias.offset;
  rel.bias = static_cast<const uint8_t*>(ex.bias);
  rel.bias_stride_b = ex.bias_stride_b;
  rel.bias_stride_h = ex.bias_stride_h;
  rel.bias_f32 = ex.bias_f32;
  if (D <= 64) return bf16 ? launch_decode_best<64, true>(prm, rel, B, Sk, shared_kv, num_sms, device, stream)
                           : launch_decode_best<64, false>(prm, rel, B, Sk, shared_kv, num_sms, device, stream);
  return bf16 ? launch_decode_best<128, true>(prm, rel, B, Sk, shared_kv, num_sms, device, stream)
              : launch_decode_best<128, false>(prm, rel, B, Sk, shared_kv, num_sms, device, stream);
}

}  // namespace fo

extern "C" int64_t fo_rel_attn_workspace(int H, int Sq, int Sk, const int* starts, int n_starts, int two_sided,
                                         int query_offset, int64_t bias_rows) {
  fo::clear_error();
  RelArgs rel;
  if (make_rel_args(&rel, H, Sq, Sk, starts, n_starts, two_sided, query_offset)) return -1;
  if (H <= 0 || bias_rows < 0) {
    fo::fail(FO_ERR_INVALID_ARGUMENT, "H must be positive and bias_rows not negative (got %d %lld)", H, (long long)bias_rows);
    return -1;
  }
  return expanded_bytes(rel.bias, H, bias_rows, Sk);
}

extern "C" int64_t fo_rel_attn_bwd_workspace(int B, int H, int Sq, int Sk, int D, int num_buckets, int dropout) {
  fo::clear_error();
  if (B <= 0 || H <= 0 || Sq <= 0 || Sk <= 0 || D <= 0 || num_buckets <= 0) {
    fo::fail(FO_ERR_INVALID_ARGUMENT, "B, H, Sq, Sk, D and num_buckets must be positive");
    return -1;
  }
  return (tile_sum_floats(B, H, Sq, Sk, D, dropout != 0) + bucket_sum_floats(B, H, Sk, D, num_buckets, dropout != 0)) * 4;
}

extern "C" int fo_rel_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                               int B, int H, int Sq, int Sk, int D,
                               const int64_t q_strides[3], const int64_t k_strides[3],
                               const int64_t v_strides[3], const int64_t o_strides[3],
                               int dtype, int causal, float softmax_scale,
                               const void* table, const int64_t table_strides[2], int table_dtype,
                               const int* starts, int n_starts, int two_sided, int query_offset, void* workspace,
                               const void* bias, const int64_t bias_strides[3], int bias_dtype,
                               float dropout_p, uint64_t rng_seed, uint64_t rng_offset,
                               int device, void* stream) {
  fo::clear_error();
  RelArgs rel;
  if (int rc = make_rel_args(&rel, H, Sq, Sk, starts, n_starts, two_sided, query_offset)) return rc;
  if (int rc = set_table(&rel, table, table_dtype, table_strides, dtype)) return rc;
  if (int rc = check_bias_strides(bias, bias_strides)) return rc;
  fo::AttnExtras ex;
  if (int rc = fo::make_attn_extras(&ex, bias, bias_strides, bias_dtype, dtype, dropout_p, rng_seed, rng_offset)) return rc;
  // one query row without an LSE: the decoding kernel finds the buckets by itself
  if (int rc = set_expanded(&rel, workspace, ex, B, H, Sk, Sq > 1 || lse != nullptr || ex.dropout)) return rc;
  return fo::attn_fwd_impl(q, k, v, o, lse, B, H, Sq, Sk, D, q_strides, k_strides, v_strides, o_strides, dtype, causal,
                           softmax_scale, &ex, &rel, device, stream);
}

extern "C" int fo_rel_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout,
                               const float* lse, void* dq, void* dk, void* dv, void* dtable, float* dq_accum, float* delta,
                               float* partials, int B, int H, int Sq, int Sk, int D,
                               const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                               const int64_t o_strides[3], const int64_t do_strides[3],
                               const int64_t dq_strides[3], const int64_t dk_strides[3], const int64_t dv_strides[3],
                               int dtype, int causal, float softmax_scale, int table_dtype,
                               const int* starts, int n_starts, int two_sided, int query_offset, const void* workspace,
                               const void* bias, const int64_t bias_strides[3], int bias_dtype,
                               float dropout_p, uint64_t rng_seed, uint64_t rng_offset,
                               int device, void* stream) {
  fo::clear_error();
  RelArgs rel;
  // the table itself is not read again: its expanded form, in the workspace, is
  if (int rc = make_rel_args(&rel, H, Sq, Sk, starts, n_starts, two_sided, query_offset)) return rc;
  if (int rc = check_table_dtype(table_dtype, dtype)) return rc;
  FO_REQUIRE(dtable == nullptr || partials != nullptr, "the table's gradient needs its workspace");
  FO_REQUIRE((reinterpret_cast<uintptr_t>(partials) & 7) == 0, "partials must be 8-byte aligned");
  FO_REQUIRE(reinterpret_cast<uintptr_t>(dtable) % (table_dtype == FO_F32 ? 4 : 2) == 0, "dtable is not aligned to its elements");
  if (int rc = check_bias_strides(bias, bias_strides)) return rc;
  fo::AttnExtras ex;
  if (int rc = fo::make_attn_extras(&ex, bias, bias_strides, bias_dtype, dtype, dropout_p, rng_seed, rng_offset)) return rc;
  if (int rc = set_expanded(&rel, const_cast<void*>(workspace), ex, B, H, Sk, true)) return rc;
  rel.dtable = dtable;
  rel.table_dtype = table_dtype;
  if (dtable != nullptr) {
    FO_REQUIRE(4LL * B * ((Sq + fo::kBlockM - 1) / fo::kBlockM) < (1LL << 31) &&
                   1LL * B * ((Sk + fo::kBlockN - 1) / fo::kBlockN) * 16 < (1LL << 31),
               "too many tiles for the table's gradient");
    rel.bias.tile_sums = reinterpret_cast<float2*>(partials);
    rel.bias.acc = partials + tile_sum_floats(B, H, Sq, Sk, D, ex.dropout != 0);
  }
  if (int rc = fo::attn_bwd_impl(q, k, v, o, dout, lse, dq, dk, dv, dq_accum, delta, B, H, Sq, Sk, D, q_strides, k_strides,
                                 v_strides, o_strides, do_strides, dq_strides, dk_strides, dv_strides, dtype, causal,
                                 softmax_scale, &ex, &rel, device, stream))
    return rc;
  return FO_OK;
}
