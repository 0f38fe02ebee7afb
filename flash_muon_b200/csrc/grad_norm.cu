// Norm over all gradients of a model, the factor that clips it, and the scaling by it.  Each is one
// pass over the gradients: the bound is HBM.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>
#include <vector>

#include "common.cuh"

namespace fm {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;         // elements a block takes at a time
constexpr int kSmallTable = 64;      // tensors of one launch: the table travels as a kernel argument
constexpr int kLargeTable = 1024;
// Up to 256 units of 1024 elements, a unit per warp at a time, go to one cluster of blocks, which adds up
// in shared memory and leaves the result itself: one launch instead of two, 2 us less host time.  On the device
// that is 2.5 us instead of 3.0 for 2^16 bf16 elements, 2.8 instead of 3.2 for 2^17, 3.6 instead of 3.3 for 2^18,
// 5.4 instead of 3.4 for 2^19.
constexpr int kUnit = 1024, kMaxUnits = 256, kCluster = 8, kClusterThreads = 512;
// Scaling walks with up to 128 blocks per SM.  A block per tile would be faster where there is something
// to do (353 M bf16 elements: 209 instead of 222 us), but within the norm, as most steps are, its
// 172,000 blocks take 93 us to find that out, these 13 to 18.
constexpr int kScaleThreads = 128, kScaleTile = 2048, kScaleBlocks = 128;
constexpr int kMaxBlocks = 1184;     // partial sums of one launch, 8 per SM; fixed, so that the
                                     // order of the sum is the same whatever else runs

template <int N>
struct Table {
  void* g[N];
  long long n[N];
  unsigned first[N + 1];  // first chunk of each tensor; [count] is their number
  uint8_t dtype[N];       // fm_dtype
  int count;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// Tensor of a chunk, found by every thread for itself in constant memory.
template <typename Tab>
__device__ __forceinline__ int find(const Tab& tab, unsigned chunk) {
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Blocks walk contiguous ranges of the chunks (of `chunk` elements) of all tensors.
template <typename Tab, typename Body>
__device__ __forceinline__ void walk(const Tab& tab, int chunk, Body body) {
  const unsigned total = tab.first[tab.count];
  const unsigned lo = (unsigned)((unsigned long long)total * blockIdx.x / gridDim.x);
  const unsigned hi = (unsigned)((unsigned long long)total * (blockIdx.x + 1) / gridDim.x);
  int at = find(tab, lo);
  for (unsigned c = lo; c < hi; ++c) {
    while (tab.first[at + 1] <= c) ++at;
    const long long base = (long long)(c - tab.first[at]) * chunk, left = tab.n[at] - base;
    const int len = (int)(left < chunk ? left : chunk);
    switch (tab.dtype[at]) {
      case FM_BF16: body(static_cast<__nv_bfloat16*>(tab.g[at]) + base, len); break;
      case FM_F16: body(static_cast<__half*>(tab.g[at]) + base, len); break;
      default: body(static_cast<float*>(tab.g[at]) + base, len); break;
    }
  }
}

// Sum of squares of a chunk: at most 32 squares per thread in fp32.
template <typename T>
__device__ __forceinline__ float chunk_sumsq(const T* g, int len) {
  constexpr int V = 16 / sizeof(T);
  float s = 0.f;
  if (len == kChunk && (reinterpret_cast<uintptr_t>(g) & 15u) == 0) {
    constexpr int L = kChunk / (V * kThreads);
    uint4 raw[L];
#pragma unroll
    for (int i = 0; i < L; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(g) + i * kThreads + threadIdx.x);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float f = to_f<T>(e[j]);
        s = fmaf(f, f, s);
      }
    }
    return s;
  }
#pragma unroll 8
  for (int i = threadIdx.x; i < len; i += kThreads) {
    const float f = to_f<T>(g[i]);
    s = fmaf(f, f, s);
  }
  return s;
}

// Bound by HBM: 353 M bf16 elements in 289 tensors 107 us (6.6 TB/s), f32 203 us (7.0 TB/s).  Blocks walk, for
// few partial sums; a warp's loads of a chunk go out together.
template <int N>
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ Table<N> tab, double* partials) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  double s = 0.0;
  walk(tab, kChunk, [&](auto* g, int len) { s += (double)chunk_sumsq(g, len); });
  s = warp_sum(s);
  __shared__ double red[kThreads / 32];
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = red[0];
    for (int i = 1; i < kThreads / 32; ++i) s += red[i];
    partials[blockIdx.x] = s;
  }
}

__device__ __forceinline__ void write_result(double sum, double max_norm, float* result) {
  const float norm = (float)sqrt(sum);
  const float ratio = (float)max_norm / (norm + 1e-6f);
  result[0] = norm;
  result[1] = fabsf(norm) <= 3.402823466e38f ? fminf(ratio, 1.f) : __int_as_float(0x7fc00000);
}

// Sum of a lane's 32 squares of a unit of `len` elements.
template <typename T>
__device__ __forceinline__ float unit_sumsq(const T* g, int len) {
  constexpr int V = 16 / sizeof(T), L = kUnit / (32 * V);
  const int lane = threadIdx.x & 31;
  float s = 0.f;
  if (len == kUnit && (reinterpret_cast<uintptr_t>(g) & 15u) == 0) {
    uint4 raw[L];
#pragma unroll
    for (int i = 0; i < L; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(g) + i * 32 + lane);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float f = to_f<T>(e[j]);
        s = fmaf(f, f, s);
      }
    }
    return s;
  }
#pragma unroll 8
  for (int i = lane; i < len; i += 32) {
    const float f = to_f<T>(g[i]);
    s = fmaf(f, f, s);
  }
  return s;
}

// Bound by latency: 97 vectors of 1024 in one launch, 8.0 to 9.1 us a call with its host side (two launches 10.7).
template <int N>
__global__ void __cluster_dims__(kCluster) __launch_bounds__(kClusterThreads)
grad_norm_small_kernel(const __grid_constant__ Table<N> tab, double max_norm, float* result) {
  namespace cg = cooperative_groups;
  __shared__ double red[kClusterThreads / 32], all[kCluster];
  const cg::cluster_group cluster = cg::this_cluster();
  // A block's shared memory may be written from outside only once the block runs: all say so here, and
  // the wait stands in front of the write, behind the loads.
  cluster.barrier_arrive();
  const unsigned total = tab.first[tab.count];
  const int warp = threadIdx.x >> 5;
  double s = 0.0;
  for (unsigned u = warp * kCluster + blockIdx.x; u < total; u += kCluster * (kClusterThreads / 32)) {
    const int at = find(tab, u);
    const long long base = (long long)(u - tab.first[at]) * kUnit, left = tab.n[at] - base;
    const int len = (int)(left < kUnit ? left : kUnit);
    switch (tab.dtype[at]) {
      case FM_BF16: s += (double)unit_sumsq(static_cast<__nv_bfloat16*>(tab.g[at]) + base, len); break;
      case FM_F16: s += (double)unit_sumsq(static_cast<__half*>(tab.g[at]) + base, len); break;
      default: s += (double)unit_sumsq(static_cast<float*>(tab.g[at]) + base, len); break;
    }
  }
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) red[warp] = s;
  __syncthreads();
  cluster.barrier_wait();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kClusterThreads / 32; ++i) s += red[i];
    cluster.map_shared_rank(all, 0)[blockIdx.x] = s;
  }
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    s = all[0];
    for (int i = 1; i < kCluster; ++i) s += all[i];
    write_result(s, max_norm, result);
  }
}

__global__ void __launch_bounds__(kThreads)
grad_norm_result_kernel(const double* partials, int count, double max_norm, float* result) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) s += partials[i];
  s = warp_sum(s);
  __shared__ double red[kThreads / 32];
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = red[0];
    for (int i = 1; i < kThreads / 32; ++i) s += red[i];
    write_result(s, max_norm, result);
  }
}

// A tile of 2048 elements, 16 per thread.
template <typename T>
__device__ __forceinline__ void scale_tile(T* g, int len, float f) {
  if (len == kScaleTile && (reinterpret_cast<uintptr_t>(g) & 15u) == 0) {
    constexpr int L = sizeof(T);  // 16-byte accesses of a thread, kScaleThreads apart
    constexpr int V = 16 / sizeof(T);
    uint4 raw[L];
#pragma unroll
    for (int i = 0; i < L; ++i) raw[i] = reinterpret_cast<const uint4*>(g)[i * kScaleThreads + threadIdx.x];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      T* e = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = from_f<T>(to_f<T>(e[j]) * f);
      reinterpret_cast<uint4*>(g)[i * kScaleThreads + threadIdx.x] = raw[i];
    }
    return;
  }
#pragma unroll 8
  for (int i = threadIdx.x; i < len; i += kScaleThreads) g[i] = from_f<T>(to_f<T>(g[i]) * f);
}

template <int N>
__global__ void __launch_bounds__(kScaleThreads)
scale_multi_kernel(const __grid_constant__ Table<N> tab, const float* factor) {
  const float f = *factor;
  if (f == 1.f) return;
  walk(tab, kScaleTile, [&](auto* g, int len) { scale_tile(g, len, f); });
}

int check_tensors(const void* const* grads, const int64_t* numels, const int32_t* dtypes, int count) {
  if (count < 0) return fail(FM_ERR_INVALID, "negative tensor count");
  if (count > 0 && (!grads || !numels || !dtypes)) return fail(FM_ERR_INVALID, "null table");
  for (int i = 0; i < count; ++i) {
    if (numels[i] < 0 || numels[i] > (int64_t)1 << 38) return fail(FM_ERR_INVALID, "bad element count at %d", i);
    if (dtypes[i] < FM_BF16 || dtypes[i] > FM_F32) return fail(FM_ERR_UNSUPPORTED, "unknown dtype %d", dtypes[i]);
    if (numels[i] == 0) continue;
    if (!grads[i] || reinterpret_cast<uintptr_t>(grads[i]) % dtype_bytes(dtypes[i]) != 0)
      return fail(FM_ERR_INVALID, "null or misaligned tensor pointer at %d", i);
  }
  return FM_OK;
}

// Refuses tensors that share memory, also with the factor: two blocks would scale it, once or twice.
int check_apart(void* const* grads, const int64_t* numels, const int32_t* dtypes, int count, const float* factor) {
  std::vector<std::pair<uintptr_t, uintptr_t>> r;
  r.reserve(count + 1);
  r.emplace_back((uintptr_t)factor, (uintptr_t)factor + 4);
  for (int i = 0; i < count; ++i)
    if (numels[i] > 0)
      r.emplace_back((uintptr_t)grads[i], (uintptr_t)grads[i] + (size_t)numels[i] * dtype_bytes(dtypes[i]));
  if (!std::is_sorted(r.begin(), r.end())) std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i].first < r[i - 1].second) return fail(FM_ERR_INVALID, "tensors to scale overlap (the same one twice?)");
  return FM_OK;
}

// Fills tables and hands each to `go(table)`.
template <int N, typename Go>
int for_tables(const void* const* grads, const int64_t* numels, const int32_t* dtypes, int count, int chunk, Go go) {
  Table<N> tab;
  tab.count = 0;
  tab.first[0] = 0;
  for (int i = 0; i < count; ++i) {
    if (numels[i] == 0) continue;
    const long long chunks = (numels[i] + chunk - 1) / chunk;
    if (tab.count == N || tab.first[tab.count] + chunks > 0x7fffffffLL) {
      const int rc = go(tab);
      if (rc != FM_OK) return rc;
      tab.count = 0;
    }
    tab.g[tab.count] = const_cast<void*>(grads[i]);
    tab.n[tab.count] = numels[i];
    tab.dtype[tab.count] = (uint8_t)dtypes[i];
    tab.first[tab.count + 1] = tab.first[tab.count] + (unsigned)chunks;
    ++tab.count;
  }
  return tab.count > 0 ? go(tab) : FM_OK;
}

// A launch ends when its table is full or the next tensor's chunks (at most 2^25) would overflow the
// 31 bits of the chunk count, so it holds 63 tensors at least.
int most_launches(int count) { return count / 63 + 1; }

}  // namespace
}  // namespace fm

extern "C" size_t fm_grad_norm_workspace_bytes(int count) {
  if (count < 0) return 0;
  return (size_t)fm::kMaxBlocks * fm::most_launches(count) * sizeof(double);
}

extern "C" int fm_grad_norm(const void* const* grads, const int64_t* numels, const int32_t* dtypes, int count,
                            double max_norm, float* result, void* workspace, size_t workspace_bytes,
                            void* stream) {
  using namespace fm;
  clear_error();
  int rc = check_tensors(grads, numels, dtypes, count);
  if (rc != FM_OK) return rc;
  if (!result || (reinterpret_cast<uintptr_t>(result) & 3u) != 0) return fail(FM_ERR_INVALID, "null or misaligned result");
  if (!(max_norm >= 0.0)) return fail(FM_ERR_INVALID, "max_norm must not be negative");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0)
    return fail(FM_ERR_INVALID, "null or misaligned workspace");
  if (workspace_bytes < fm_grad_norm_workspace_bytes(count)) return fail(FM_ERR_WORKSPACE, "workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* partials = static_cast<double*>(workspace);
  int used = 0;
  auto go = [&](const auto& tab) -> int {
    const unsigned total = tab.first[tab.count];
    const unsigned blocks = total < (unsigned)kMaxBlocks ? total : (unsigned)kMaxBlocks;
    grad_norm_kernel<<<blocks, kThreads, 0, st>>>(tab, partials + used);
    used += (int)blocks;
    FM_CUDA_CHECK(cudaGetLastError());
    return FM_OK;
  };
  long long units = 0;
  for (int i = 0; i < count; ++i) units += (numels[i] + kUnit - 1) / kUnit;
  if (units > 0 && units <= kMaxUnits) {
    auto all = [&](const auto& tab) -> int {
      grad_norm_small_kernel<<<kCluster, kClusterThreads, 0, st>>>(tab, max_norm, result);
      FM_CUDA_CHECK(cudaGetLastError());
      return FM_OK;
    };
    // every tensor that is not empty has a unit: one table holds them all
    return units <= kSmallTable ? for_tables<kSmallTable>(grads, numels, dtypes, count, kUnit, all)
                                : for_tables<kMaxUnits>(grads, numels, dtypes, count, kUnit, all);
  }
  rc = count <= kSmallTable ? for_tables<kSmallTable>(grads, numels, dtypes, count, kChunk, go)
                            : for_tables<kLargeTable>(grads, numels, dtypes, count, kChunk, go);
  if (rc != FM_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = used > 0 && options().pdl != 0 ? 1 : 0;
  FM_CUDA_CHECK(cudaLaunchKernelEx(&cfg, grad_norm_result_kernel, (const double*)partials, used, max_norm, result));
  return FM_OK;
}

extern "C" int fm_scale_multi(void* const* grads, const int64_t* numels, const int32_t* dtypes, int count,
                              const float* factor, void* stream) {
  using namespace fm;
  clear_error();
  int rc = check_tensors(grads, numels, dtypes, count);
  if (rc != FM_OK) return rc;
  if (!factor || (reinterpret_cast<uintptr_t>(factor) & 3u) != 0) return fail(FM_ERR_INVALID, "null or misaligned factor");
  try {
    rc = check_apart(grads, numels, dtypes, count, factor);
  } catch (...) {
    rc = fail(FM_ERR_INVALID, "out of host memory");
  }
  if (rc != FM_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](const auto& tab) -> int {
    const unsigned total = tab.first[tab.count];
    const unsigned most = (unsigned)sm_count() * kScaleBlocks;
    scale_multi_kernel<<<total < most ? total : most, kScaleThreads, 0, st>>>(tab, factor);
    FM_CUDA_CHECK(cudaGetLastError());
    return FM_OK;
  };
  return count <= kSmallTable ? for_tables<kSmallTable>(grads, numels, dtypes, count, kScaleTile, go)
                              : for_tables<kLargeTable>(grads, numels, dtypes, count, kScaleTile, go);
}
