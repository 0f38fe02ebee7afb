// AdamW over many tensors in one launch, states in fp32 or in 8 bits (state8.cuh).
//
// For a parameter w with gradient g, factor s, moments m and v and step count t (counted from 1):
//   g' = s g;  m <- b1 m + (1 - b1) g';  v <- b2 v + (1 - b2) g'^2
//   w <- w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// all in fp32, w rounded once where it is stored in 16 bits; with a master copy w is the master and
// the parameter its rounded value.  1 - b^t and its root are formed in 64 bits (at t = 1 and
// b2 = 0.999 fp32 would leave 1 - b2^t four digits).
//
// Every element is independent and read and written once: the bound is HBM.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "common.cuh"
#include "state8.cuh"

namespace fm {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;       // elements a block takes at a time; a tensor's last chunk is short
constexpr int kMaxHyper = 8;       // parameter groups of one launch
constexpr int kSmallTable = 40;    // tensors of one launch: the table travels as a kernel argument,
constexpr int kLargeTable = 360;   // small (4 KB) where it suffices, else up to the limit of 32764 bytes
constexpr int kCountTable = 480;

struct Entry {
  void* p;
  const void* g;
  float* w;          // master copy or null
  void* m;
  void* v;
  uint8_t* ms;       // exponent bytes, 8-bit states only
  uint8_t* vs;
  const float* step;
  long long n;
  uint32_t seed;
  uint16_t hyper;
  uint16_t vec;      // every pointer allows 16-byte accesses
};
struct Hyper {
  double lr, beta1, beta2;
  const float* lr_dev;  // overrides lr where set
  float eps, wd;
};
template <int N>
struct Table {
  Entry e[N];
  unsigned first[N + 1];  // first chunk of each tensor; [count] is their number
  Hyper h[kMaxHyper];
  const float* scale;
  int count;
};
struct CountTable {
  float* step[kCountTable];
  const float* scale;
  int count;
};

struct Coef {
  float b1, omb1, b2, omb2, eps, decay, size, root;
  uint32_t key;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// N elements from / to a 16-byte aligned address
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* src, T (&dst)[N]) {
#pragma unroll
  for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i)
    reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* dst, const T (&src)[N]) {
#pragma unroll
  for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i)
    reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
}

__device__ __forceinline__ double power(double b, unsigned t) {
  double r = 1.0;
  for (; t != 0; t >>= 1) {
    if (t & 1u) r *= b;
    b *= b;
  }
  return r;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// A step whose factor is not finite (the norm it came from was not) is not taken at all.
__device__ __forceinline__ bool skipped(const float* scale) { return scale != nullptr && !finite(*scale); }

__device__ __forceinline__ Coef coefficients(const Hyper& h, const Entry& e) {
  const unsigned t = (unsigned)*e.step;
  const double lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
  Coef c;
  c.b1 = (float)h.beta1;
  c.omb1 = (float)(1.0 - h.beta1);
  c.b2 = (float)h.beta2;
  c.omb2 = (float)(1.0 - h.beta2);
  c.eps = h.eps;
  c.decay = (float)(1.0 - lr * (double)h.wd);
  c.size = (float)(lr / (1.0 - power(h.beta1, t)));
  c.root = (float)(1.0 / sqrt(1.0 - power(h.beta2, t)));
  c.key = state8::step_key(e.seed, t);
  return c;
}

__device__ __forceinline__ void moments(const Coef& c, float g, float& m, float& v) {
  m = fmaf(c.b1, m, c.omb1 * g);
  v = fmaf(c.b2, v, c.omb2 * (g * g));
}

// ---------------------------------------------------------------- step counts
// The counts are advanced by a launch of their own ahead of the step's: every block of the step
// reads its tensor's count, so none of them may write it.
__global__ void __launch_bounds__(kThreads) adamw_count_kernel(const __grid_constant__ CountTable tab) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (skipped(tab.scale)) return;
  for (int i = threadIdx.x; i < tab.count; i += kThreads) *tab.step[i] += 1.f;
}

// Blocks of a step walk contiguous ranges of the chunks of all tensors.  `body(entry, base, coef)` does
// one chunk.
template <typename Tab, typename Body>
__device__ __forceinline__ void walk(const Tab& tab, Body body) {
  __shared__ int s_at;
  __shared__ Coef s_coef;
  const unsigned total = tab.first[tab.count];
  const unsigned lo = (unsigned)((unsigned long long)total * blockIdx.x / gridDim.x);
  const unsigned hi = (unsigned)((unsigned long long)total * (blockIdx.x + 1) / gridDim.x);
  for (int i = threadIdx.x; i < tab.count; i += kThreads)
    if (tab.first[i] <= lo && lo < tab.first[i + 1]) s_at = i;
  // the counts of this step are the previous launch's
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (skipped(tab.scale)) return;
  const float scale = tab.scale ? *tab.scale : 1.f;
  __syncthreads();
  int at = s_at;
  Coef coef;
  for (unsigned c = lo; c < hi;) {
    __syncthreads();
    if (threadIdx.x == 0) s_coef = coefficients(tab.h[tab.e[at].hyper], tab.e[at]);
    __syncthreads();
    coef = s_coef;
    const unsigned first = tab.first[at], end = min(tab.first[at + 1], hi);
    for (; c < end; ++c) body(tab.e[at], (long long)(c - first) * kChunk, coef, scale);
    ++at;
  }
}

// ---------------------------------------------------------------- states in fp32
template <typename P, typename G, bool kMaster, int N>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(const __grid_constant__ Table<N> tab) {
  walk(tab, [](const Entry& e, long long base, const Coef& c, float scale) {
    P* const p = static_cast<P*>(e.p);
    const G* const g = static_cast<const G*>(e.g);
    float* const m = static_cast<float*>(e.m);
    float* const v = static_cast<float*>(e.v);
    auto update = [&](float w, float gr, float& mm, float& vv) {
      moments(c, gr * scale, mm, vv);
      return fmaf(w, c.decay, -c.size * (mm / fmaf(sqrtf(vv), c.root, c.eps)));
    };
    if (e.vec && base + kChunk <= e.n) {
#pragma unroll
      for (int i = 0; i < kChunk / (8 * kThreads); ++i) {
        const long long at = base + (i * kThreads + threadIdx.x) * 8;
        alignas(16) P pv[8];
        alignas(16) G gv[8];
        alignas(16) float mv[8], vv[8], wv[8];
        if (kMaster) load_vec(e.w + at, wv);
        else load_vec(p + at, pv);
        load_vec(g + at, gv);
        load_vec(m + at, mv);
        load_vec(v + at, vv);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = update(kMaster ? wv[j] : to_f<P>(pv[j]), to_f<G>(gv[j]), mv[j], vv[j]);
          if (kMaster) wv[j] = w;
          pv[j] = from_f<P>(w);
        }
        store_vec(p + at, pv);
        if (kMaster) store_vec(e.w + at, wv);
        store_vec(m + at, mv);
        store_vec(v + at, vv);
      }
      return;
    }
    const long long end = min(base + kChunk, e.n);
#pragma unroll 4
    for (long long at = base + threadIdx.x; at < end; at += kThreads) {
      float mm = m[at], vv = v[at];
      const float w = update(kMaster ? e.w[at] : to_f<P>(p[at]), to_f<G>(g[at]), mm, vv);
      p[at] = from_f<P>(w);
      if (kMaster) e.w[at] = w;
      m[at] = mm;
      v[at] = vv;
    }
  });
}

// ---------------------------------------------------------------- states in 8 bits
// A thread takes 16 consecutive elements, two neighbouring lanes a block of 32.
__device__ __forceinline__ uint32_t finite_max(const float (&x)[16]) {
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) mx = max(mx, __float_as_uint(x[j]) & 0x7fffffffu);
  if (mx >= 0x7f800000u) {  // an element that is not finite does not set the block's exponent
    mx = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t u = __float_as_uint(x[j]) & 0x7fffffffu;
      if (u < 0x7f800000u) mx = max(mx, u);
    }
  }
  return max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
}

template <typename P, typename G, bool kMaster, int N>
__global__ void __launch_bounds__(kThreads, 2) adamw8_kernel(const __grid_constant__ Table<N> tab) {
  walk(tab, [](const Entry& e, long long base, const Coef& c, float scale) {
    P* const p = static_cast<P*>(e.p);
    const G* const g = static_cast<const G*>(e.g);
    const long long at = base + threadIdx.x * 16;
    const long long left = e.n - at;                       // elements of this thread's 16 that exist
    const bool in = at < (e.n + 31) / 32 * 32;             // its block does
    const bool full = left >= 16;
    uint8_t* const mc = static_cast<uint8_t*>(e.m) + at;
    uint8_t* const vc = static_cast<uint8_t*>(e.v) + at;
    alignas(16) uint8_t mq[16], vq[16];
    int mb = 127, vb = 127;
    alignas(16) float w[16];
    alignas(16) P pv[16];
    alignas(16) G gv[16];
    if (in) {
      *reinterpret_cast<uint4*>(mq) = *reinterpret_cast<const uint4*>(mc);
      *reinterpret_cast<uint4*>(vq) = *reinterpret_cast<const uint4*>(vc);
      mb = e.ms[at >> 5];
      vb = e.vs[at >> 5];
    } else {
      *reinterpret_cast<uint4*>(mq) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(vq) = make_uint4(0, 0, 0, 0);
    }
    if (full && e.vec) {
      load_vec(g + at, gv);
      if (kMaster) load_vec(e.w + at, w);
      else load_vec(p + at, pv);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const bool here = j < left;
        gv[j] = here ? g[at + j] : from_f<G>(0.f);
        if (kMaster) w[j] = here ? e.w[at + j] : 0.f;
        else pv[j] = here ? p[at + j] : from_f<P>(0.f);
      }
    }
    float m[16], v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const bool here = full || j < left;  // bytes behind the last element count as zeros
      m[j] = here ? state8::decode_m(mq[j], mb) : 0.f;
      v[j] = here ? state8::decode_v(vq[j], vb) : 0.f;
      moments(c, to_f<G>(gv[j]) * scale, m[j], v[j]);
      if (!kMaster) w[j] = to_f<P>(pv[j]);
      // the update takes the moments before they are rounded to 8 bits
      w[j] = fmaf(w[j], c.decay, -c.size * (m[j] / fmaf(sqrtf(v[j]), c.root, c.eps)));
      pv[j] = from_f<P>(w[j]);
    }
    mb = state8::block_exp(finite_max(m), state8::kMinExpM);
    vb = state8::block_exp(finite_max(v), state8::kMinExpV);
    const uint32_t key = state8::index_key(c.key, (uint32_t)(at >> 32));
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t h = state8::random_bits(key, (uint32_t)at + j);
      mq[j] = state8::encode_m(m[j], mb, state8::random_m(h));
      vq[j] = state8::encode_v(v[j], vb, state8::random_v(h));
    }
    if (!in) return;
    *reinterpret_cast<uint4*>(mc) = *reinterpret_cast<uint4*>(mq);
    *reinterpret_cast<uint4*>(vc) = *reinterpret_cast<uint4*>(vq);
    if ((threadIdx.x & 1) == 0) {
      e.ms[at >> 5] = (uint8_t)mb;
      e.vs[at >> 5] = (uint8_t)vb;
    }
    if (full && e.vec) {
      store_vec(p + at, pv);
      if (kMaster) store_vec(e.w + at, w);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j < left) {
          p[at + j] = pv[j];
          if (kMaster) e.w[at + j] = w[j];
        }
      }
    }
  });
}

// ---------------------------------------------------------------- 8-bit states to values and back
template <typename T>
__global__ void __launch_bounds__(kThreads)
adamw8_values_kernel(const uint8_t* codes, const uint8_t* exps, long long n, int moment, T* out) {
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kThreads) {
    const int b = exps[i >> 5];
    out[i] = from_f<T>(moment == 1 ? state8::decode_m(codes[i], b) : state8::decode_v(codes[i], b));
  }
}

// One warp per block of 32, rounding to nearest.
template <typename T>
__global__ void __launch_bounds__(kThreads)
adamw8_encode_kernel(const T* values, long long n, int moment, uint8_t* codes, uint8_t* exps) {
  const long long padded = (n + 31) / 32 * 32;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < padded;
       i += (long long)gridDim.x * kThreads) {
    const float x = i < n ? to_f<T>(values[i]) : 0.f;
    uint32_t mx = __float_as_uint(x) & 0x7fffffffu;
    if (mx >= 0x7f800000u) mx = 0;
    mx = __reduce_max_sync(0xffffffffu, mx);
    const int b = state8::block_exp(mx, moment == 1 ? state8::kMinExpM : state8::kMinExpV);
    codes[i] = moment == 1 ? state8::encode_m(x, b, state8::kNearest) : state8::encode_v(x, b, state8::kNearest);
    if ((threadIdx.x & 31) == 0) exps[i >> 5] = (uint8_t)b;
  }
}

// ---------------------------------------------------------------- host side
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

struct Range {
  uintptr_t begin, end;
  bool written;
};

// Refuses a call whose written memory overlaps anything else of the call: two threads would race.
int check_ranges(std::vector<Range>& r) {
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;
  for (const Range& x : r) {
    if (x.begin < (x.written ? any : written))
      return fail(FM_ERR_INVALID, "tensors of the step overlap (the same parameter twice?)");
    any = std::max(any, x.end);
    if (x.written) written = std::max(written, x.end);
  }
  return FM_OK;
}

int check_group(const fm_adamw_group& g, int gi, std::vector<Range>& ranges) {
  if (g.count < 0) return fail(FM_ERR_INVALID, "group %d: negative count", gi);
  if (g.count == 0) return FM_OK;
  if (!g.params || !g.grads || !g.exp_avg || !g.exp_avg_sq || !g.steps || !g.numels)
    return fail(FM_ERR_INVALID, "group %d: null array", gi);
  if (g.state_bits != 32 && g.state_bits != 8)
    return fail(FM_ERR_UNSUPPORTED, "group %d: states have 32 or 8 bits, not %d", gi, g.state_bits);
  if (g.state_bits == 8 && (!g.exp_avg_scale || !g.exp_avg_sq_scale || !g.seeds))
    return fail(FM_ERR_INVALID, "group %d: 8-bit states need scales and seeds", gi);
  if (g.p_dtype < FM_BF16 || g.p_dtype > FM_F32 || g.g_dtype < FM_BF16 || g.g_dtype > FM_F32)
    return fail(FM_ERR_UNSUPPORTED, "group %d: unknown dtype", gi);
  if (g.p_dtype != FM_F32 && g.g_dtype != g.p_dtype && g.g_dtype != FM_F32)
    return fail(FM_ERR_UNSUPPORTED, "group %d: 16-bit parameters take gradients of their own type or f32", gi);
  if (g.masters && g.p_dtype == FM_F32)
    return fail(FM_ERR_UNSUPPORTED, "group %d: f32 parameters have no master copies", gi);
  if (!aligned(g.lr_device, 4)) return fail(FM_ERR_INVALID, "group %d: misaligned lr", gi);
  if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0))
    return fail(FM_ERR_INVALID, "group %d: betas must lie in [0, 1)", gi);
  if (!(g.eps >= 0.0) || !std::isfinite(g.eps) || !std::isfinite(g.weight_decay) || !std::isfinite(g.lr))
    return fail(FM_ERR_INVALID, "group %d: lr, eps and weight_decay must be finite, eps not negative", gi);
  const size_t pb = dtype_bytes(g.p_dtype), gb = dtype_bytes(g.g_dtype), sb = g.state_bits == 8 ? 1 : 4;
  for (int i = 0; i < g.count; ++i) {
    const int64_t n = g.numels[i];
    if (n < 0 || n > (int64_t)1 << 38) return fail(FM_ERR_INVALID, "group %d: bad element count at %d", gi, i);
    if (!g.steps[i] || !aligned(g.steps[i], 4)) return fail(FM_ERR_INVALID, "group %d: bad step count at %d", gi, i);
    ranges.push_back({(uintptr_t)g.steps[i], (uintptr_t)g.steps[i] + 4, true});
    if (n == 0) continue;
    if (!g.params[i] || !g.grads[i] || !g.exp_avg[i] || !g.exp_avg_sq[i] || (g.masters && !g.masters[i]))
      return fail(FM_ERR_INVALID, "group %d: null tensor pointer at %d", gi, i);
    if (!aligned(g.params[i], pb) || !aligned(g.grads[i], gb) || (g.masters && !aligned(g.masters[i], 4)) ||
        !aligned(g.exp_avg[i], g.state_bits == 8 ? 16 : 4) || !aligned(g.exp_avg_sq[i], g.state_bits == 8 ? 16 : 4))
      return fail(FM_ERR_INVALID, "group %d: misaligned tensor at %d", gi, i);
    const size_t ns = g.state_bits == 8 ? (size_t)(n + 31) / 32 * 32 : (size_t)n;
    auto add = [&](const void* q, size_t bytes, bool written) {
      ranges.push_back({(uintptr_t)q, (uintptr_t)q + bytes, written});
    };
    add(g.params[i], n * pb, true);
    add(g.grads[i], n * gb, false);
    add(g.exp_avg[i], ns * sb, true);
    add(g.exp_avg_sq[i], ns * sb, true);
    if (g.masters) add(g.masters[i], n * 4, true);
    if (g.state_bits == 8) {
      if (!g.exp_avg_scale[i] || !g.exp_avg_sq_scale[i])
        return fail(FM_ERR_INVALID, "group %d: null scales at %d", gi, i);
      add(g.exp_avg_scale[i], ns / 32, true);
      add(g.exp_avg_sq_scale[i], ns / 32, true);
    }
  }
  return FM_OK;
}

// What a launch is compiled for.
struct Kind {
  int p, g, bits;
  bool master;
  bool operator==(const Kind& o) const { return p == o.p && g == o.g && bits == o.bits && master == o.master; }
};
Kind kind_of(const fm_adamw_group& g) { return {g.p_dtype, g.g_dtype, g.state_bits, g.masters != nullptr}; }

template <auto kernel, typename Tab>
int launch_table(const Tab& tab, bool dependent, cudaStream_t stream) {
  static int resident = 0;  // blocks per SM of this kernel
  if (resident == 0) {
    int per_sm = 0;
    FM_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, 0));
    resident = per_sm > 0 ? per_sm : 1;
  }
  const long long most = (long long)resident * sm_count();
  const long long total = tab.first[tab.count];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(total < most ? total : most));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  FM_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, tab));
  return FM_OK;
}

template <typename P, typename G, bool kMaster, int N>
int launch_kind(const Table<N>& tab, int bits, bool dependent, cudaStream_t stream) {
  if (bits == 8) return launch_table<adamw8_kernel<P, G, kMaster, N>>(tab, dependent, stream);
  return launch_table<adamw_kernel<P, G, kMaster, N>>(tab, dependent, stream);
}

template <int N>
int launch(const Table<N>& tab, const Kind& k, bool dependent, cudaStream_t st) {
  using B = __nv_bfloat16;
  using H = __half;
  if (k.p == FM_F32) {
    if (k.g == FM_F32) return launch_kind<float, float, false>(tab, k.bits, dependent, st);
    if (k.g == FM_BF16) return launch_kind<float, B, false>(tab, k.bits, dependent, st);
    return launch_kind<float, H, false>(tab, k.bits, dependent, st);
  }
  if (k.p == FM_BF16) {
    if (k.g == FM_BF16)
      return k.master ? launch_kind<B, B, true>(tab, k.bits, dependent, st)
                      : launch_kind<B, B, false>(tab, k.bits, dependent, st);
    return k.master ? launch_kind<B, float, true>(tab, k.bits, dependent, st)
                    : launch_kind<B, float, false>(tab, k.bits, dependent, st);
  }
  if (k.g == FM_F16)
    return k.master ? launch_kind<H, H, true>(tab, k.bits, dependent, st)
                    : launch_kind<H, H, false>(tab, k.bits, dependent, st);
  return k.master ? launch_kind<H, float, true>(tab, k.bits, dependent, st)
                  : launch_kind<H, float, false>(tab, k.bits, dependent, st);
}

// Collects tensors of one kind and sends them out when the table is full.
struct Batch {
  Table<kLargeTable> tab;
  Kind kind;
  int hypers = 0, last_group = -1;
  bool dependent = false;  // the next launch follows the counts directly
  cudaStream_t stream;

  int flush() {
    if (tab.count == 0) return FM_OK;
    int rc;
    if (tab.count <= kSmallTable) {
      Table<kSmallTable> small;
      std::copy(tab.e, tab.e + tab.count, small.e);
      std::copy(tab.first, tab.first + tab.count + 1, small.first);
      std::copy(tab.h, tab.h + hypers, small.h);
      small.scale = tab.scale;
      small.count = tab.count;
      rc = launch(small, kind, dependent, stream);
    } else {
      rc = launch(tab, kind, dependent, stream);
    }
    tab.count = 0;
    hypers = 0;
    last_group = -1;
    dependent = false;
    return rc;
  }

  int add(const fm_adamw_group& g, int gi, int i) {
    const int64_t n = g.numels[i];
    const int64_t chunks = (n + kChunk - 1) / kChunk;
    if (tab.count > 0 && (tab.count == kLargeTable || (last_group != gi && hypers == kMaxHyper) ||
                          tab.first[tab.count] + chunks > 0x7fffffffLL)) {
      const int rc = flush();
      if (rc != FM_OK) return rc;
    }
    if (tab.count == 0) tab.first[0] = 0;
    if (last_group != gi) {
      Hyper& h = tab.h[hypers++];
      h.lr = g.lr; h.beta1 = g.beta1; h.beta2 = g.beta2; h.lr_dev = g.lr_device;
      h.eps = (float)g.eps; h.wd = (float)g.weight_decay;
      last_group = gi;
    }
    Entry& e = tab.e[tab.count];
    e.p = g.params[i]; e.g = g.grads[i];
    e.w = g.masters ? static_cast<float*>(g.masters[i]) : nullptr;
    e.m = g.exp_avg[i]; e.v = g.exp_avg_sq[i];
    e.ms = g.state_bits == 8 ? static_cast<uint8_t*>(g.exp_avg_scale[i]) : nullptr;
    e.vs = g.state_bits == 8 ? static_cast<uint8_t*>(g.exp_avg_sq_scale[i]) : nullptr;
    e.step = g.steps[i];
    e.n = n;
    e.seed = g.state_bits == 8 ? g.seeds[i] : 0;
    e.hyper = (uint16_t)(hypers - 1);
    e.vec = aligned(e.p, 16) && aligned(e.g, 16) && aligned(e.w, 16) && aligned(e.m, 16) && aligned(e.v, 16);
    tab.first[tab.count + 1] = tab.first[tab.count] + (unsigned)chunks;
    ++tab.count;
    return FM_OK;
  }
};

int count_steps(const fm_adamw_group* groups, int ngroups, const float* scale, cudaStream_t stream) {
  CountTable tab;
  tab.scale = scale;
  tab.count = 0;
  auto flush = [&]() -> int {
    if (tab.count == 0) return FM_OK;
    adamw_count_kernel<<<1, kThreads, 0, stream>>>(tab);
    tab.count = 0;
    FM_CUDA_CHECK(cudaGetLastError());
    return FM_OK;
  };
  for (int gi = 0; gi < ngroups; ++gi) {
    for (int i = 0; i < groups[gi].count; ++i) {
      tab.step[tab.count++] = groups[gi].steps[i];
      if (tab.count == kCountTable) {
        const int rc = flush();
        if (rc != FM_OK) return rc;
      }
    }
  }
  return flush();
}

int adamw_step(const fm_adamw_group* groups, int ngroups, const float* scale, cudaStream_t stream) {
  std::vector<Range> ranges;
  size_t tensors = 0;
  for (int gi = 0; gi < ngroups; ++gi) tensors += groups[gi].count > 0 ? groups[gi].count : 0;
  ranges.reserve(tensors * 8);
  for (int gi = 0; gi < ngroups; ++gi) {
    const int rc = check_group(groups[gi], gi, ranges);
    if (rc != FM_OK) return rc;
  }
  if (tensors == 0) return FM_OK;
  if (!aligned(scale, 4)) return fail(FM_ERR_INVALID, "misaligned gradient scale");
  int rc = check_ranges(ranges);
  if (rc != FM_OK) return rc;
  rc = count_steps(groups, ngroups, scale, stream);
  if (rc != FM_OK) return rc;
  Batch batch;
  batch.tab.count = 0;
  batch.tab.scale = scale;
  batch.stream = stream;
  batch.dependent = options().pdl != 0;
  std::vector<char> done(ngroups, 0);
  for (int gi = 0; gi < ngroups; ++gi) {
    if (done[gi]) continue;
    batch.kind = kind_of(groups[gi]);
    for (int gj = gi; gj < ngroups; ++gj) {
      if (done[gj] || !(kind_of(groups[gj]) == batch.kind)) continue;
      done[gj] = 1;
      for (int i = 0; i < groups[gj].count; ++i) {
        if (groups[gj].numels[i] == 0) continue;
        rc = batch.add(groups[gj], gj, i);
        if (rc != FM_OK) return rc;
      }
    }
    rc = batch.flush();
    if (rc != FM_OK) return rc;
  }
  return FM_OK;
}

int simple_grid(long long n) {
  const long long want = (n + kThreads - 1) / kThreads, most = (long long)sm_count() * 8;
  return (int)(want < most ? want : most);
}

int check_moment(const void* a, const void* b, const void* c, int64_t n, int moment) {
  if (n < 0) return fail(FM_ERR_INVALID, "negative element count");
  if (moment != 1 && moment != 2) return fail(FM_ERR_INVALID, "moment must be 1 or 2");
  if (n > 0 && (!a || !b || !c)) return fail(FM_ERR_INVALID, "null pointer");
  return FM_OK;
}

}  // namespace
}  // namespace fm

extern "C" int fm_adamw_step(const fm_adamw_group* groups, int ngroups, const float* grad_scale, void* stream) {
  using namespace fm;
  clear_error();
  if (ngroups < 0 || (ngroups > 0 && !groups)) return fail(FM_ERR_INVALID, "bad group list");
  try {
    return adamw_step(groups, ngroups, grad_scale, static_cast<cudaStream_t>(stream));
  } catch (...) {
    return fail(FM_ERR_INVALID, "out of host memory");
  }
}

extern "C" int fm_adamw8_values(const void* codes, const void* scales, int64_t n, int moment, void* out,
                                int out_dtype, void* stream) {
  using namespace fm;
  clear_error();
  int rc = check_moment(codes, scales, out, n, moment);
  if (rc != FM_OK) return rc;
  if (out_dtype < FM_BF16 || out_dtype > FM_F32) return fail(FM_ERR_UNSUPPORTED, "unknown dtype %d", out_dtype);
  if (n == 0) return FM_OK;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = simple_grid(n);
  if (out_dtype == FM_F32)
    adamw8_values_kernel<float><<<grid, kThreads, 0, st>>>(c, s, n, moment, static_cast<float*>(out));
  else if (out_dtype == FM_BF16)
    adamw8_values_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(c, s, n, moment, static_cast<__nv_bfloat16*>(out));
  else
    adamw8_values_kernel<__half><<<grid, kThreads, 0, st>>>(c, s, n, moment, static_cast<__half*>(out));
  FM_CUDA_CHECK(cudaGetLastError());
  return FM_OK;
}

extern "C" int fm_adamw8_encode(const void* values, int v_dtype, int64_t n, int moment, void* codes, void* scales,
                                void* stream) {
  using namespace fm;
  clear_error();
  int rc = check_moment(values, codes, scales, n, moment);
  if (rc != FM_OK) return rc;
  if (v_dtype < FM_BF16 || v_dtype > FM_F32) return fail(FM_ERR_UNSUPPORTED, "unknown dtype %d", v_dtype);
  if (n == 0) return FM_OK;
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = simple_grid(n);
  if (v_dtype == FM_F32)
    adamw8_encode_kernel<float><<<grid, kThreads, 0, st>>>(static_cast<const float*>(values), n, moment, c, s);
  else if (v_dtype == FM_BF16)
    adamw8_encode_kernel<__nv_bfloat16>
        <<<grid, kThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(values), n, moment, c, s);
  else
    adamw8_encode_kernel<__half><<<grid, kThreads, 0, st>>>(static_cast<const __half*>(values), n, moment, c, s);
  FM_CUDA_CHECK(cudaGetLastError());
  return FM_OK;
}
