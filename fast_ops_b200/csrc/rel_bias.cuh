// A learned relative position bias: the score of query i and key j gets table[bucket(j - i - offset)][head].
//
// Buckets are given by the smallest distance of each of them, `starts` (0 = starts[0] <= starts[1] ...): a
// distance n lies in the last bucket whose start is not above n.  One-sided, n = max(i + offset - j, 0);
// two-sided, n = |j - i - offset|, and the keys behind the query have a second set of buckets.
//
// The tile kernels read the bias of a head as a vector over the relative position d = j - i - offset, at
// x = d + zero, divided by the softmax scale: it is added to Q K^T, and the scale in the exponent applies to both.
// It is constant from -far_left down and from far_right up, so that only the tiles near the diagonal read it at
// all; its ends reach kRelMargin further, which is more than a warp's part of such a tile can.  A thread reads neighbouring values from a place of its own, 16 bytes at a time:
// the vector is there four times, copy s shifted by s values, so that one of them is aligned for it
// (64 values by 16 loads instead of 64).  The copies are 8 banks apart, so that from shared memory eight
// threads read 32 banks; a vector too long for four copies there is kept in two.
//
// A vector bias beside it (key padding, as a rule) is brought into the same form, one row for each
// batch and head that has its own, with what lets the kernels pass over most of it: the end of the keys that
// are not masked, behind which nothing is computed, and the 64-key steps from the first value that is not 0 to
// the last one before that end.
#pragma once

#include <cstdint>

namespace fo {

constexpr int kRelMaxStarts = 256;  // buckets of one side: they travel in kernel arguments
constexpr int kRelMargin = 104;

struct RelBuckets {
  int starts[kRelMaxStarts];
  int n;          // buckets of one side
  int two_sided;
};

__device__ __forceinline__ int rel_bucket(const RelBuckets& bk, int d) {
  const int n = bk.two_sided ? abs(d) : max(-d, 0);
  int lo = 0, hi = bk.n - 1;  // starts[lo] <= n, and nothing above hi is
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (bk.starts[mid] <= n) lo = mid;
    else hi = mid - 1;
  }
  return bk.two_sided && d > 0 ? lo + bk.n : lo;
}

// A bias times `factor` (log2(e), or 1 / scale), where -1e6 and less masks as -inf does.  (Taken as a number,
// a mask that leaves a row without keys would give it an LSE of that size, from which the backward
// cannot tell P: at -1e9 the spacing of fp32 is 64, and P = exp(s - LSE) could be anything, infinity
// included.  Rows with a key left do not change: e^-1e6 is 0.)
__device__ __forceinline__ float scaled_or_masked(float v, float factor) {
  return v <= -1e6f ? __int_as_float(0xff800000) : v * factor;
}

// What the tile kernels need; null `values`: no relative bias.
struct RelBias {
  const float* values;   // [H][4][stride]: copy s holds value x + s at x
  const int* bucket_of;  // [width]
  // Backward, null without a gradient of the table: the tiles near the diagonal summed by bucket,
  // [B*H][key tiles][warps][buckets], and the sums of dS and of P over each warp's part of every tile,
  // [B*H][query tiles][key tiles][warps].
  float* acc;
  float2* tile_sums;
  int width, zero, stride;
  int smem_copies;           // copies that the kernel with the vector in shared memory keeps (2 or 4)
  const float* vec;          // [rows][rel_vec_width], or null without a vector bias
  const int4* vec_extent;    // [rows]: (keys up to the last one not masked, first step with a bias, step after the last, 0)
  int vec_row_b, vec_row_h;  // row of (b, h): b * vec_row_b + h * vec_row_h
  int vec_width;
  int far_left, far_right;
  int offset;
  int num_buckets;
};

// Where a rectangle of scores lies whose relative positions go from `first` to `last`.
enum RelSide { kRelNear = 0, kRelLeft = 1, kRelRight = 2 };
__device__ __forceinline__ RelSide rel_side(const RelBias& rel, int first, int last) {
  return last <= -rel.far_left ? kRelLeft : first >= rel.far_right ? kRelRight : kRelNear;
}

// Bias (divided by the softmax scale) of relative position d for head h, whatever d is.  (This and the row's extent
// below are not read as constant data, __ldg: a kernel whose launch overlaps the expansion starts before they are
// written.)
__device__ __forceinline__ float rel_value(const RelBias& rel, int h, int d) {
  const int x = min(max(d, -rel.zero), rel.width - 1 - rel.zero) + rel.zero;
  return __ldcg(rel.values + static_cast<int64_t>(h) * 4 * rel.stride + x);
}

// Row of the vector bias, and the keys that a head computes: `keys`, or those up to the last one not masked, but
// at least one (whose score is -inf if it is masked too).
__device__ __forceinline__ int64_t rel_vec_row(const RelBias& rel, int b, int h) {
  return static_cast<int64_t>(b) * rel.vec_row_b + static_cast<int64_t>(h) * rel.vec_row_h;
}
__device__ __forceinline__ int rel_keys(const RelBias& rel, int b, int h, int keys) {
  return rel.vec == nullptr ? keys : min(keys, max(__ldcg(&rel.vec_extent[rel_vec_row(rel, b, h)].x), 1));
}

// Keys of a row of `vec`: whole key tiles.
__host__ __device__ inline int rel_vec_width(int Sk) { return (Sk + 127) / 128 * 128; }

// Adds 32 values of a bias, in shared memory or not, to 32 scores that are still to be scaled.
template <bool kShared>
__device__ __forceinline__ void add_rel_bias(uint32_t (&s)[32], const float4* bias) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 r = kShared ? bias[i] : __ldg(bias + i);
    const float2 lo = __fadd2_rn(make_float2(__uint_as_float(s[4 * i]), __uint_as_float(s[4 * i + 1])), make_float2(r.x, r.y));
    const float2 hi = __fadd2_rn(make_float2(__uint_as_float(s[4 * i + 2]), __uint_as_float(s[4 * i + 3])), make_float2(r.z, r.w));
    s[4 * i] = __float_as_uint(lo.x);
    s[4 * i + 1] = __float_as_uint(lo.y);
    s[4 * i + 2] = __float_as_uint(hi.x);
    s[4 * i + 3] = __float_as_uint(hi.y);
  }
}

// The same from an 8-byte aligned place in shared memory.
__device__ __forceinline__ void add_rel_bias_pairs(uint32_t (&s)[32], const float2* bias) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 x = __fadd2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), bias[i]);
    s[2 * i] = __float_as_uint(x.x);
    s[2 * i + 1] = __float_as_uint(x.y);
  }
}

// Where a thread finds the values from x on (x >= 0): 16-byte aligned, for head h.
__device__ __forceinline__ const float4* rel_vector(const RelBias& rel, int h, int x) {
  const int s = x & 3;
  return reinterpret_cast<const float4*>(rel.values + (static_cast<int64_t>(h) * 4 + s) * rel.stride + (x - s));
}

}  // namespace fo
