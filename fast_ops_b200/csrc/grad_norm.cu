// The 2-norm over all elements of a list of gradients, and the factor that clips them to a norm:
//
//   norm = sqrt(sum_t sum_i g_t[i]^2)      coef = min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM: every gradient is read once.  The tensor list travels in the kernel's arguments (no device
// table, nothing cached, nothing allocated), so a call can be captured into a graph the first time it is made.
//
// A thread squares and sums eight fp32 elements in fp32 and adds each such sum to a double, so that what the
// norm loses to rounding does not grow with the list; where the fp32 sum of eight leaves the range in which its
// squares are normal numbers (gradients beyond 1e18 or all below 1e-15), the eight are summed again in
// double.  16-bit elements are summed in double throughout.  Every sum is formed in a fixed order: the same list
// gives the same bits on every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cooperative_groups.h>

#include <cmath>
#include <cstring>

#include "fo_host.h"
#include "fo_ptx.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;     // elements of one group: 16 bytes of a 16-bit type, 32 of fp32
constexpr int kUnroll = 4;  // groups of a thread in flight
constexpr int kChunk = kThreads * kVec * kUnroll;  // 8192 elements: what a block takes at a time

// Most tensors of one launch: 21 bytes each, 21.5 KB of the 32764 that kernel arguments may take.  A longer list takes
// several launches.  Short lists use the small form, whose arguments are a tenth as long.
constexpr int kMaxTensors = 1024, kFewTensors = 96;

template <int kMax>
struct TensorList {
  const void* ptr[kMax];
  int64_t numel[kMax];
  uint32_t first_chunk[kMax + 1];  // index of the tensor's first chunk among all chunks of the launch
  uint8_t dtype[kMax];
  int n;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Eight elements from a 16-byte aligned address.
__device__ __forceinline__ void load8(const float* p, float (&v)[kVec]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[kVec]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[kVec]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 h;
    memcpy(&h, &w[i], 4);
    const float2 f = __half22float2(h);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Eight squares in double, for what fp32 does not hold: zeros, tiny or huge values, infinities and NaN.
__device__ __forceinline__ double squares_in_double(const float (&v)[kVec]) {
  double d = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) d += static_cast<double>(v[i]) * static_cast<double>(v[i]);
  return d;
}

// fp32 values: eight squares are summed in fp32, whose roundings have no preferred sign here.
__device__ __forceinline__ double sum_of_squares8(const float (&v)[kVec], const float*) {
  const float s = ((v[0] * v[0] + v[1] * v[1]) + (v[2] * v[2] + v[3] * v[3])) +
                  ((v[4] * v[4] + v[5] * v[5]) + (v[6] * v[6] + v[7] * v[7]));
  return s > 1e-30f && s < 1e37f ? static_cast<double>(s) : squares_in_double(v);
}

// 16-bit values: their squares are exact in fp32 but end in zeros, so that sums of two are often halfway between two
// fp32 numbers and always rounded down there (6e-9 of the sum in bf16, 1e-8 in fp16, whatever the length of the
// list).  They are added in double, to which a square goes by its bits: the exponent's bias changes by 896, and the
// mantissa (at most 22 bits of 24) moves three places.  (By conversions, 16 a clock and SM, the norm of 2^28 bf16
// elements takes 95.5 us instead of 93 with the second launch; in fp32 88.5.)
template <class T>
__device__ __forceinline__ double sum_of_squares8(const float (&v)[kVec], const T*) {
  uint32_t bits[kVec], most = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    bits[i] = __float_as_uint(v[i] * v[i]);
    most = max(most, bits[i] - 0x00800000u);  // zeros and subnormal numbers wrap around
  }
  if (most >= 0x7f000000u) return squares_in_double(v);  // one of them, an infinity or NaN is among the squares
  double d = 0, e = 0;
#pragma unroll
  for (int i = 0; i < kVec; i += 2) {
    d += __hiloint2double((bits[i] >> 3) + 0x38000000u, bits[i] << 29);
    e += __hiloint2double((bits[i + 1] >> 3) + 0x38000000u, bits[i + 1] << 29);
  }
  return d + e;
}

// This thread's share of one chunk's sum: `left` elements of the tensor remain from `p` on.
template <typename T>
__device__ __forceinline__ double chunk_sum(const T* p, int64_t left) {
  double sum = 0;
  if (left >= kChunk && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    float v[kUnroll][kVec];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) load8(p + (u * kThreads + threadIdx.x) * kVec, v[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) sum += sum_of_squares8(v[u], p);
  } else {
    // the tail of a tensor, or one whose storage is not 16-byte aligned
    const int n = left < kChunk ? static_cast<int>(left) : kChunk;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const double x = static_cast<double>(load1(p + i));
      sum += x * x;
    }
  }
  return sum;
}

// Sum over the block's threads, valid in thread 0; `scratch` holds one value per warp.
__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = threadIdx.x < kThreads / 32 ? scratch[threadIdx.x] : 0;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  }
  return v;
}

// The calling thread's share of the chunks first, first + step, ... of a list.
template <int kMax>
__device__ __forceinline__ double list_sum(const TensorList<kMax>& list, uint32_t first, uint32_t step) {
  const uint32_t total = list.first_chunk[list.n];
  int t = 0;
  double sum = 0;
  for (uint32_t chunk = first; chunk < total; chunk += step) {
    while (chunk >= list.first_chunk[t + 1]) ++t;  // a block's chunks only go up
    const int64_t base = static_cast<int64_t>(chunk - list.first_chunk[t]) * kChunk;
    const int64_t left = list.numel[t] - base;
    const int dtype = list.dtype[t];
    if (dtype == FO_F32) sum += chunk_sum(static_cast<const float*>(list.ptr[t]) + base, left);
    else if (dtype == FO_BF16) sum += chunk_sum(static_cast<const __nv_bfloat16*>(list.ptr[t]) + base, left);
    else sum += chunk_sum(static_cast<const __half*>(list.ptr[t]) + base, left);
  }
  return sum;
}

// Where a call's results go (null: not wanted).
struct Results {
  double* sumsq;
  float* norm;
  float* coef;
  double max_norm;
};

__device__ __forceinline__ void store_results(const Results& out, double sum) {
  if (out.sumsq != nullptr) *out.sumsq = sum;
  const double root = sqrt(sum);
  const float norm = static_cast<float>(root);
  if (out.norm != nullptr) *out.norm = norm;
  if (out.coef != nullptr) {
    // In fp32, as clipping in memory by the norm that is reported.  Finite gradients can have a norm beyond fp32; by
    // the infinity that is reported they would all become 0, so they are scaled by the root in double.
    const float coef = isinf(norm) ? static_cast<float>(out.max_norm / root)
                                   : __fdiv_rn(static_cast<float>(out.max_norm), __fadd_rn(norm, 1e-6f));
    *out.coef = coef > 1.f ? 1.f : coef;  // a NaN stays one
  }
}

// partials[block] = the block's share of the sum of squares.
template <int kMax>
__global__ void __launch_bounds__(kThreads)
grad_sumsq_kernel(const __grid_constant__ TensorList<kMax> list, double* __restrict__ partials) {
  __shared__ double scratch[kThreads / 32];
  fo::grid_allow_next();
  const double sum = block_sum(list_sum(list, blockIdx.x, gridDim.x), scratch);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// A short list in one launch: a cluster of blocks, the first of which adds up what the others have.  Back to back in a
// graph, bf16, this and the two launches: 8192 elements 2.6 and 2.8 us, 65536 2.8 and 3.2, 131072 3.6 and 3.4, 262144
// (32 chunks) 4.9 and 3.0; the host saves the 2.5 us of a launch.
constexpr int kClusterBlocks = 8;
constexpr uint32_t kClusterChunks = 2 * kClusterBlocks;

__global__ void __cluster_dims__(kClusterBlocks, 1, 1) __launch_bounds__(kThreads)
grad_norm_small_kernel(const __grid_constant__ TensorList<kFewTensors> list, const Results out) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double scratch[kThreads / 32];
  __shared__ double block_total;
  const double sum = block_sum(list_sum(list, blockIdx.x, kClusterBlocks), scratch);
  if (threadIdx.x == 0) block_total = sum;
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double total = 0;
    for (int c = 0; c < kClusterBlocks; ++c) total += *cluster.map_shared_rank(&block_total, c);
    store_results(out, total);
  }
  cluster.sync();  // no block leaves while its shared memory is being read
}

// One block: the sum of all partials, and the results from it.
__global__ void __launch_bounds__(kThreads)
grad_norm_finish_kernel(const double* __restrict__ partials, int n, const Results out) {
  __shared__ double scratch[kThreads / 32];
  double sum = 0;
  fo::grid_wait_previous();  // its launch overlaps the kernel that writes the partials
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += kThreads) sum += __ldcg(partials + i);
  sum = block_sum(sum, scratch);
  if (threadIdx.x == 0) store_results(out, sum);
}

// Blocks of the widest launch, and doubles of workspace for each launch.  Several rounds of resident blocks (five
// per SM) even out their ends: 2^28 elements with 5 / 8 / 16 / 32 / 64 blocks per SM, bf16 94.6 / 96.4 / 94.5 / 93.1 /
// 95.1 us, fp32 161 / 155 / 155.5 / 155.7 / 154.3 (with the second launch).
constexpr int kMaxBlocks = 148 * 32;

// The tensors begin to end - 1 that are not empty.
template <int kMax>
void fill_list(TensorList<kMax>* list, const void* const* grads, const int64_t* numels, const int* dtypes, int begin, int end) {
  int n = 0;
  uint32_t chunks = 0;
  for (int i = begin; i < end; ++i) {
    if (numels[i] == 0) continue;
    list->ptr[n] = grads[i];
    list->numel[n] = numels[i];
    list->dtype[n] = static_cast<uint8_t>(dtypes[i]);
    list->first_chunk[n] = chunks;
    chunks += static_cast<uint32_t>((numels[i] + kChunk - 1) / kChunk);
    ++n;
  }
  list->first_chunk[n] = chunks;
  list->n = n;
}

template <int kMax>
int launch_sumsq(const void* const* grads, const int64_t* numels, const int* dtypes, int begin, int end, double* partials,
                 int* blocks_out, cudaStream_t stream) {
  TensorList<kMax> list;
  fill_list(&list, grads, numels, dtypes, begin, end);
  const uint32_t chunks = list.first_chunk[list.n];
  *blocks_out = 0;
  if (chunks == 0) return FO_OK;
  const int blocks = chunks < static_cast<uint32_t>(kMaxBlocks) ? static_cast<int>(chunks) : kMaxBlocks;
  grad_sumsq_kernel<kMax><<<blocks, kThreads, 0, stream>>>(list, partials);
  fo::g_launch_count.fetch_add(1, std::memory_order_relaxed);
  FO_CUDA_CHECK(cudaGetLastError());
  *blocks_out = blocks;
  return FO_OK;
}

int launch_finish(const double* partials, int n, const Results& out, cudaStream_t stream) {
  FO_CUDA_CHECK(fo::launch_overlapping(grad_norm_finish_kernel, dim3(1), dim3(kThreads), 0, stream, partials, n, out));
  fo::g_launch_count.fetch_add(1, std::memory_order_relaxed);
  return FO_OK;
}

int check_max_norm(double max_norm) {
  FO_REQUIRE(max_norm >= 0.0, "max_norm must be non-negative (got %g)", max_norm);
  return FO_OK;
}

}  // namespace

extern "C" int64_t fo_grad_norm_workspace(int n_tensors) {
  const int64_t launches = n_tensors <= kMaxTensors ? 1 : (static_cast<int64_t>(n_tensors) + kMaxTensors - 1) / kMaxTensors;
  return launches * kMaxBlocks;
}

extern "C" int fo_grad_norm(const void* const* grads, const int64_t* numels, const int* dtypes, int n_tensors,
                            double max_norm, double* workspace, double* sumsq, float* norm, float* coef, int device,
                            void* stream) {
  fo::clear_error();
  FO_REQUIRE(n_tensors >= 0, "n_tensors must be >= 0");
  FO_REQUIRE(n_tensors == 0 || (grads && numels && dtypes), "null tensor list");
  FO_REQUIRE(workspace != nullptr, "null workspace");
  FO_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "workspace must be 8-byte aligned");
  FO_REQUIRE(sumsq || norm || coef, "nowhere to put the result");
  if (int rc = check_max_norm(max_norm)) return rc;
  int64_t total = 0;
  for (int i = 0; i < n_tensors; ++i) {
    FO_REQUIRE(numels[i] >= 0, "tensor %d has negative numel", i);
    FO_REQUIRE(numels[i] == 0 || grads[i] != nullptr, "tensor %d has a null pointer", i);
    FO_REQUIRE(dtypes[i] == FO_F16 || dtypes[i] == FO_BF16 || dtypes[i] == FO_F32, "tensor %d: bad dtype %d", i, dtypes[i]);
    FO_REQUIRE(numels[i] == 0 || reinterpret_cast<uintptr_t>(grads[i]) % (dtypes[i] == FO_F32 ? 4 : 2) == 0,
               "tensor %d is not aligned to its elements", i);
    FO_REQUIRE(numels[i] <= (int64_t{1} << 44), "tensor %d is too large", i);
    total += (numels[i] + kChunk - 1) / kChunk;
  }
  FO_REQUIRE(total < (int64_t{1} << 31), "the list has too many elements");
  fo::DeviceGuard guard(device);
  FO_REQUIRE(guard.ok, "cannot make device %d current", device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Results out{sumsq, norm, coef, max_norm};
  if (n_tensors <= kFewTensors && total <= kClusterChunks) {
    TensorList<kFewTensors> list;
    fill_list(&list, grads, numels, dtypes, 0, n_tensors);
    grad_norm_small_kernel<<<kClusterBlocks, kThreads, 0, s>>>(list, out);
    fo::g_launch_count.fetch_add(1, std::memory_order_relaxed);
    FO_CUDA_CHECK(cudaGetLastError());
    return FO_OK;
  }
  int used = 0;  // partials written so far
  for (int begin = 0; begin < n_tensors; begin += kMaxTensors) {
    const int end = n_tensors - begin < kMaxTensors ? n_tensors : begin + kMaxTensors;
    int blocks = 0;
    const int rc = end - begin <= kFewTensors
                       ? launch_sumsq<kFewTensors>(grads, numels, dtypes, begin, end, workspace + used, &blocks, s)
                       : launch_sumsq<kMaxTensors>(grads, numels, dtypes, begin, end, workspace + used, &blocks, s);
    if (rc) return rc;
    used += blocks;
  }
  return launch_finish(workspace, used, out, s);
}

extern "C" int fo_grad_norm_finish(const double* sumsq, double max_norm, float* norm, float* coef, int device, void* stream) {
  fo::clear_error();
  FO_REQUIRE(sumsq != nullptr && (norm || coef), "null pointer");
  if (int rc = check_max_norm(max_norm)) return rc;
  fo::DeviceGuard guard(device);
  FO_REQUIRE(guard.ok, "cannot make device %d current", device);
  return launch_finish(sumsq, 1, Results{nullptr, norm, coef, max_norm}, static_cast<cudaStream_t>(stream));
}
