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
#include <type_traits>
#include <vector>

#include "common.cuh"
#include "state8.cuh"

namespace fm {
namespace {

constexpr int kThreads = 128;
constexpr int kEach32 = 8;         // elements per thread with 32-bit states: a tile of 1024
constexpr int kMaxThreads = 512;   // of a block that takes a whole small tensor
constexpr int kPart8 = 2048;       // 16 per thread with 8-bit states, where two threads share a block of
constexpr int kMaxParts = 8;       // 32, and a block takes up to 8 such parts
constexpr int kWholeParts = 2;     // parts of a whole small tensor
constexpr int kMaxHyper = 8;       // parameter groups of one launch
// Tensors of one launch.  The table travels as a kernel argument, of 3, 9 or 30 KB (the limit is 32764
// bytes): the largest costs the host 1.4 us more per launch than the smallest.
constexpr int kSmallTable = 24, kMediumTable = 96, kLargeTable = 360;
constexpr int kCountTable = 480;

struct Entry {
  void* p;
  const void* g;
  float* w;          // master copy or null
  void* m;
  void* v;
  uint8_t* ms;       // exponent bytes, 8-bit states only
  uint8_t* vs;
  float* step;
  long long n;
  uint32_t seed;
  uint16_t hyper;
  uint16_t vec;      // every pointer allows the widest accesses made (16-byte codes, 32 bytes else)
};
struct Hyper {
  double lr, beta1, beta2, wd;
  const float* lr_dev;            // overrides lr where set
  float b1, omb1, b2, omb2, eps;  // betas, 1 - betas
  float root_omb2;
};
template <int N>
struct Table {
  Entry e[N];
  unsigned first[N + 1];  // first tile of each tensor; [count] is their number
  Hyper h[kMaxHyper];
  const float* scale;
  int count;
  int parts;              // 8-bit states: parts of a tile
  int threads;            // 32-bit states: threads of a block
  int whole;              // every tensor has one block, which advances its count
};
struct CountTable {
  float* step[kCountTable];
  const float* scale;
  int count;
};

// What depends on a tensor's step count.
struct Coef {
  float size, root, decay;  // lr / (1 - b1^t), sqrt(1 - b2^t), 1 - lr wd
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

// N elements from / to an address aligned to 32 bytes (16 where they are no more): 32 bytes per
// access where possible.  Two 16-byte stores per thread would each write half of every sector.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* src, T (&dst)[N]) {
  constexpr int kBytes = N * sizeof(T);
  if constexpr (kBytes % 32 == 0) {
    uint32_t* d = reinterpret_cast<uint32_t*>(dst);
#pragma unroll
    for (int i = 0; i < kBytes / 32; ++i)
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(d[8 * i]), "=r"(d[8 * i + 1]), "=r"(d[8 * i + 2]), "=r"(d[8 * i + 3]), "=r"(d[8 * i + 4]),
                     "=r"(d[8 * i + 5]), "=r"(d[8 * i + 6]), "=r"(d[8 * i + 7])
                   : "l"(reinterpret_cast<const char*>(src) + 32 * i)
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* dst, const T (&src)[N]) {
  constexpr int kBytes = N * sizeof(T);
  if constexpr (kBytes % 32 == 0) {
    const uint32_t* d = reinterpret_cast<const uint32_t*>(src);
#pragma unroll
    for (int i = 0; i < kBytes / 32; ++i)
      asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(d[8 * i]), "r"(d[8 * i + 1]),
                   "r"(d[8 * i + 2]), "r"(d[8 * i + 3]), "r"(d[8 * i + 4]), "r"(d[8 * i + 5]), "r"(d[8 * i + 6]),
                   "r"(d[8 * i + 7]), "l"(reinterpret_cast<char*>(dst) + 32 * i)
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i)
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
  }
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

// Tensor of a tile.  Every thread searches for itself: the table is in constant memory, all lanes
// read the same word, and no barrier stands before the loads of the tile.  The first tensors, where
// the large ones mostly are, are found in the fewest steps (an embedding followed by 65 norms: 426 us,
// so 423).
template <typename Tab>
__device__ __forceinline__ int find(const Tab& tab, unsigned tile) {
  int lo = 0, hi = 1;
  while (hi < tab.count && tab.first[hi] <= tile) {
    lo = hi;
    hi *= 2;
  }
  hi = min(hi, tab.count);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= tile) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The coefficients of the block's tensor, one per warp's first thread, behind the loads of its tile:
// reading the count and the powers (17 dependent 64-bit products at t = 100000) take less than the
// loads do.
__device__ __forceinline__ void coefficients(const Hyper& h, const Entry& e, uint32_t index_hi, bool whole, bool taken,
                                             Coef* c) {
  // the counts are the previous launch's
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float count = 0.f;
  if ((threadIdx.x & 31) == 0) {
    count = *reinterpret_cast<const volatile float*>(e.step) + (whole ? 1.f : 0.f);
    const unsigned t = (unsigned)count;
    const int which = threadIdx.x >> 5;
    if (which == 0) {
      const float lr = h.lr_dev ? *h.lr_dev : (float)h.lr;
      c->size = lr / (float)(1.0 - power(h.beta1, t));
    } else if (which == 1) {
      c->root = sqrtf((float)(1.0 - power(h.beta2, t)));
    } else if (which == 2) {
      c->key = state8::index_key(state8::step_key(e.seed, t), index_hi);
    } else if (which == 3) {
      c->decay = (float)(1.0 - (h.lr_dev ? (double)*h.lr_dev : h.lr) * h.wd);
    }
  }
  __syncthreads();
  if (whole && taken && threadIdx.x == 0) *e.step = count;  // read by all of its readers
}

// Root and reciprocal within 1 ulp.  The correctly rounded ones cost the 32-bit step 8 registers per
// thread and 1 to 2 %.  Subnormal arguments count as zero, except for sqrt_approx.
__device__ __forceinline__ float root_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---------------------------------------------------------------- step counts
// The counts are advanced by a launch of their own ahead of the step's: every block of the step
// reads its tensor's count, so none of them may write it.  The step's blocks start while it runs
// and load their tiles: all that those hold was written before this launch began.  Where all
// tensors of a kind are small a block takes each of them whole and advances its count itself.
__global__ void __launch_bounds__(kThreads) adamw_count_kernel(const __grid_constant__ CountTable tab) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (skipped(tab.scale)) return;
  for (int i = threadIdx.x; i < tab.count; i += kThreads) *tab.step[i] += 1.f;
}

// ---------------------------------------------------------------- states in fp32
// Bound by HBM: 22 bytes per bf16 element, 28 per f32 one or with a master.  A tile of 1024 elements per
// block of 128 threads: many small blocks keep loads, arithmetic and stores of different tiles mixed
// where persistent blocks ran in step (524 M f32 elements 2.68 ms, so 2.10 = 6.98 TB/s; 131 M bf16 ones
// 541 us, so 425 = 6.8 TB/s; a copy runs at 6.55).
// kWhole: a block of up to 512 threads takes a whole tensor.
template <typename P, typename G, bool kMaster, bool kWhole, int N>
__global__ void __launch_bounds__(kWhole ? kMaxThreads : kThreads) adamw_kernel(const __grid_constant__ Table<N> tab) {
  __shared__ Coef s_coef;
  const int ti = find(tab, blockIdx.x);
  const Entry& e = tab.e[ti];
  const Hyper& h = tab.h[e.hyper];
  const int threads = kWhole ? blockDim.x : kThreads, tile = threads * kEach32;
  const long long base = (long long)(blockIdx.x - tab.first[ti]) * tile;
  P* const p = static_cast<P*>(e.p) + base;
  const G* const g = static_cast<const G*>(e.g) + base;
  float* const w = e.w + base;
  float* const m = static_cast<float*>(e.m) + base;
  float* const v = static_cast<float*>(e.v) + base;
  const bool vec = e.vec && base + tile <= e.n;
  const int len = (int)(e.n - base < tile ? e.n - base : tile);
  alignas(16) P pv[8];
  alignas(16) G gv[8];
  alignas(16) float mv[8], vv[8], wv[8];
  if (vec) {  // 8 neighbouring elements
    const int at = threadIdx.x * 8;
    if (kMaster) load_vec(w + at, wv);
    else load_vec(p + at, pv);
    load_vec(g + at, gv);
    load_vec(m + at, mv);
    load_vec(v + at, vv);
  } else {    // 8 elements `threads` apart
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = j * threads + threadIdx.x;
      const bool here = at < len;
      if (kMaster) wv[j] = here ? w[at] : 0.f;
      else pv[j] = here ? p[at] : from_f<P>(0.f);
      gv[j] = here ? g[at] : from_f<G>(0.f);
      mv[j] = here ? m[at] : 0.f;
      vv[j] = here ? v[at] : 0.f;
    }
  }
  const float scale = tab.scale ? *tab.scale : 1.f;
  coefficients(h, e, 0, kWhole, finite(scale), &s_coef);
  if (!finite(scale)) return;
  // size m / (sqrt(v) / root + eps) = size root m / (sqrt(v) + eps root)
  const float decay = s_coef.decay, size = -s_coef.size * s_coef.root, eps = h.eps * s_coef.root;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float gr = to_f<G>(gv[j]) * scale;
    mv[j] = fmaf(h.b1, mv[j], h.omb1 * gr);
    vv[j] = fmaf(h.b2, vv[j], h.omb2 * (gr * gr));
    wv[j] = fmaf(kMaster ? wv[j] : to_f<P>(pv[j]), decay, size * (mv[j] * rcp_approx(sqrt_approx(vv[j]) + eps)));
    pv[j] = from_f<P>(wv[j]);
  }
  if (vec) {
    const int at = threadIdx.x * 8;
    store_vec(p + at, pv);
    if (kMaster) store_vec(w + at, wv);
    store_vec(m + at, mv);
    store_vec(v + at, vv);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = j * threads + threadIdx.x;
      if (at < len) {
        p[at] = pv[j];
        if (kMaster) w[at] = wv[j];
        m[at] = mv[j];
        v[at] = vv[j];
      }
    }
  }
}

// ---------------------------------------------------------------- states in 8 bits
// A thread takes 16 consecutive elements, two neighbouring lanes a block of 32.  The bytes of a
// step are few enough (10 per bf16 element) that instructions bound it, so arithmetic goes by pairs
// (fp32x2) and the codes are handled as floats where the hardware converts them:
//   decode m: e4m3 pairs to f16 pairs, exact; v: the code shifted to bit 7 IS an f16 number;
//   encode: scaled by the block's power of two (state8.cuh) the code is the bits above bit 20, the
//   random number is added below and cut off.
// The parts of a block's tile are copied to shared memory two ahead.  67 M bf16 elements 115 us (5.9 TB/s,
// 90 % of a copy; 46 instructions per element, issue slots 77 % busy), f32 169 us (98 %), bf16 with masters 173 us
// (96 %); elements at odd addresses 209 to 287 us (48 to 66 %).
// Two cases that hardly ever occur leave this path: a block whose largest magnitude is not finite or
// beyond what one normal fp32 factor scales, and a positive v whose code came out 0.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 both(float x) { return pack2(x, x); }
// the largest magnitude; not a number if one of them is not
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ f32x2 halves_to_floats(uint32_t h2) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
  return pack2(f.x, f.y);
}
// a half that is not a number becomes infinite, others stay
__device__ __forceinline__ uint32_t at_most_inf(uint32_t h2) {
  uint32_t r;
  asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h2), "r"(0x7c007c00u));
  return r;
}
// Codes of a word (the upper two where `upper`) read as e4m3 and f16, without their block's factor
// (state8.cuh).  Fresh states have scale byte 0 and only zero codes.
__device__ __forceinline__ f32x2 decode_m2(uint32_t w, bool upper) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((unsigned short)(upper ? w >> 16 : w)));
  return halves_to_floats(h2);
}
__device__ __forceinline__ f32x2 decode_v2(uint32_t w, bool upper) {
  // code 255, infinity, comes out of the shift as "not a number"
  return halves_to_floats(at_most_inf(__byte_perm(w, 0, upper ? 0x4342 : 0x4140) << 7));
}
// A word of padding per 16: a thread's 16 elements and a warp's neighbouring ones are both free of
// bank conflicts.
__device__ __forceinline__ int padded(int i) { return i + (i >> 4); }

// Block maxima (bit patterns) below which 2^(14 - b) and 2^(29 - b), which scale a block to its codes,
// are normal fp32 numbers: moments below 2^14 and 2^29.
constexpr uint32_t kFastMaxM = 141u << 23, kFastMaxV = 156u << 23;

// 16 bytes from global to shared memory, in the background
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// 2048 elements of type T as 16-byte chunks in shared memory.  A thread's 16 elements are 1, 2 or 4
// consecutive chunks; their low bits are exchanged with higher ones so that the eight lanes of a
// shared-memory access find eight different banks.
template <typename T>
struct Staged {
  static constexpr int kPer = sizeof(T);            // chunks per thread
  static constexpr int kChunks = kThreads * kPer;
  uint4 c[kChunks];
  __device__ static int slot(int chunk) { return kPer == 1 ? chunk : chunk ^ ((chunk >> 3) & (kPer - 1)); }
  __device__ void fetch(const T* src) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = i * kThreads + threadIdx.x;
      copy_async(&c[slot(k)], reinterpret_cast<const uint4*>(src) + k);
    }
  }
  __device__ void read(T (&dst)[16]) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) reinterpret_cast<uint4*>(dst)[i] = c[slot(threadIdx.x * kPer + i)];
  }
};

// Resident blocks per SM that registers are kept down for: 6, with two float32 arrays in shared memory 5.
// A seventh of 16-bit types leaves 72 registers, which some builds spill (114 to 132 us where 6 take 115).  16-bit
// parameters with masters and float32 gradients spill 8 bytes at 5: 67 M elements 196 us, 95 % of a copy.
template <typename W, typename G>
constexpr int resident8() {
  return sizeof(W) + sizeof(G) <= 6 ? 6 : 5;
}

template <typename P, typename G, bool kMaster, int N>
__global__ void __launch_bounds__(kThreads, resident8<std::conditional_t<kMaster, float, P>, G>()) adamw8_kernel(const __grid_constant__ Table<N> tab) {
  using W = std::conditional_t<kMaster, float, P>;  // what the weights are read from
  struct Stage {
    Staged<uint8_t> m, v;
    Staged<G> g;
    Staged<W> w;
  };
  struct Plain {  // parts that are not copied in the background
    float w[kPart8 / 16 * 17], g[kPart8 / 16 * 17];
  };
  union Shared {
    Stage stage[2];
    Plain plain;
    __device__ Shared() {}
  };
  __shared__ Shared sh;
  __shared__ Coef s_coef;
  float* const s_w = sh.plain.w;
  float* const s_g = sh.plain.g;
  const int ti = find(tab, blockIdx.x);
  const Entry& e = tab.e[ti];
  const Hyper& h = tab.h[e.hyper];
  const int tile = tab.parts * kPart8;
  const long long base = (long long)(blockIdx.x - tab.first[ti]) * tile;
  const unsigned len = (unsigned)(e.n - base < tile ? e.n - base : tile);
  const unsigned coded = (len + 31) & ~31u;  // codes of this tile
  const unsigned mine = threadIdx.x * 16;
  P* const p = static_cast<P*>(e.p) + base;
  const G* const g = static_cast<const G*>(e.g) + base;
  float* const w = e.w + base;
  uint8_t* const mc = static_cast<uint8_t*>(e.m) + base;
  uint8_t* const vc = static_cast<uint8_t*>(e.v) + base;
  uint8_t* const ms = e.ms + (base >> 5);
  uint8_t* const vs = e.vs + (base >> 5);
  const float scale = tab.scale ? *tab.scale : 1.f;

  // Whole parts of tensors whose addresses allow it arrive in shared memory two parts ahead.
  auto fetch = [&](unsigned start, int k) {
    if (e.vec && start + kPart8 <= len) {
      Stage& st = sh.stage[k];
      st.m.fetch(mc + start);
      st.v.fetch(vc + start);
      st.g.fetch(g + start);
      if constexpr (kMaster) st.w.fetch(w + start);
      else st.w.fetch(p + start);
    }
    copy_commit();
  };
  fetch(0, 0);
  fetch(kPart8, 1);
  int mb_next = 127, vb_next = 127;  // exponent bytes, a part ahead in registers
  auto fetch_exps = [&](unsigned at) {
    if (at < coded) {
      mb_next = ms[at >> 5];
      vb_next = vs[at >> 5];
    }
  };
  fetch_exps(mine);
  for (unsigned start = 0, stage = 0; start < len; start += kPart8, stage ^= 1) {
    const unsigned at = start + mine;
    const bool vec = e.vec && start + kPart8 <= len;
    alignas(16) uint8_t mq[16], vq[16];
    int mb = mb_next, vb = vb_next;
    alignas(16) W wv[16];
    alignas(16) G gv[16];
    fetch_exps(at + kPart8);
    if (vec) {
      copy_wait<1>();
      __syncthreads();
      const Stage& st = sh.stage[stage];
      st.m.read(mq);
      st.v.read(vq);
      st.g.read(gv);
      st.w.read(wv);
    } else {  // through shared memory: neighbouring threads read neighbouring elements
      *reinterpret_cast<uint4*>(mq) = *reinterpret_cast<uint4*>(vq) = make_uint4(0, 0, 0, 0);
      if (at < coded) {
        *reinterpret_cast<uint4*>(mq) = *reinterpret_cast<const uint4*>(mc + at);
        *reinterpret_cast<uint4*>(vq) = *reinterpret_cast<const uint4*>(vc + at);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const unsigned i = j * kThreads + threadIdx.x;
        s_g[padded(i)] = start + i < len ? to_f<G>(g[start + i]) : 0.f;
        s_w[padded(i)] = start + i < len ? (kMaster ? w[start + i] : to_f<P>(p[start + i])) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        gv[j] = from_f<G>(s_g[padded(mine + j)]);
        wv[j] = from_f<W>(s_w[padded(mine + j)]);
      }
      // bytes behind the last element count as zeros
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int left = (int)len - (int)at - 4 * k;
        const uint32_t keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        reinterpret_cast<uint32_t*>(mq)[k] &= keep;
        reinterpret_cast<uint32_t*>(vq)[k] &= keep;
      }
    }
    if (start == 0) {
      coefficients(h, e, (uint32_t)(base >> 32), tab.whole, finite(scale), &s_coef);
      if (!finite(scale)) {
        copy_wait<0>();
        return;
      }
    }
    // the factor of the gradient goes into the constants; that of the second moment is applied before the
    // square, which it keeps in range
    const f32x2 decay = both(s_coef.decay), size = both(-s_coef.size * s_coef.root), eps = both(h.eps * s_coef.root);
    const f32x2 b1 = both(h.b1), c1 = both(h.omb1 * scale), b2 = both(h.b2), c2 = both(h.root_omb2 * scale);

    float m[16], v[16];
    alignas(16) W wn[16];  // rounded already: half the registers for 16-bit types
    const f32x2 mf = both(state8::factor_m(mb)), vf = both(state8::factor_v(vb));
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      f32x2 m2 = mul2(decode_m2(reinterpret_cast<uint32_t*>(mq)[j / 4], j & 2), mf);
      f32x2 v2 = mul2(decode_v2(reinterpret_cast<uint32_t*>(vq)[j / 4], j & 2), vf);
      const f32x2 g2 = pack2(to_f<G>(gv[j]), to_f<G>(gv[j + 1])), u2 = mul2(c2, g2);
      m2 = fma2(b1, m2, mul2(c1, g2));
      v2 = fma2(u2, u2, mul2(b2, v2));
      unpack2(m2, m[j], m[j + 1]);
      unpack2(v2, v[j], v[j + 1]);
      // the update takes the moments before they are rounded to 8 bits
      float d0, d1;
      unpack2(add2(pack2(root_approx(v[j]), root_approx(v[j + 1])), eps), d0, d1);
      const f32x2 d2 = mul2(m2, pack2(rcp_approx(d0), rcp_approx(d1)));
      const f32x2 w2 = pack2(to_f<W>(wv[j]), to_f<W>(wv[j + 1]));
      unpack2(fma2(w2, decay, mul2(size, d2)), d0, d1);
      wn[j] = from_f<W>(d0);
      wn[j + 1] = from_f<W>(d1);
    }
    if (vec) {
      __syncthreads();  // every thread has read its elements
      fetch(start + 2 * kPart8, stage);
      if constexpr (kMaster) {
        alignas(16) P out[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) out[j] = from_f<P>(wn[j]);
        store_vec(p + at, out);
        store_vec(w + at, wn);
      } else {
        store_vec(p + at, wn);
      }
    } else {  // written from there below; a thread overwrites only what it alone has read
#pragma unroll
      for (int j = 0; j < 16; ++j) s_w[padded(mine + j)] = to_f<W>(wn[j]);
    }
    float mx = max_abs(m[0], m[1], m[2]), vx = max_abs(v[0], v[1], v[2]);
#pragma unroll
    for (int j = 3; j < 15; j += 2) {
      mx = max_abs(mx, m[j], m[j + 1]);
      vx = max_abs(vx, v[j], v[j + 1]);
    }
    uint32_t mt = __float_as_uint(max_abs(mx, m[15], 0.f)), vt = __float_as_uint(max_abs(vx, v[15], 0.f));
    mt = max(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
    vt = max(vt, __shfl_xor_sync(0xffffffffu, vt, 1));
    // mix(key ^ (index + j)) for j < 16: the index's low bits are zero, and the first xor-shift of
    // the mix does not reach j
    uint32_t key = s_coef.key ^ ((uint32_t)base + at);
    key ^= key >> 16;
    if (mt < kFastMaxM && vt < kFastMaxV) {
      mb = max((int)(mt >> 23), state8::kMinExpM);
      vb = max((int)(vt >> 23), state8::kMinExpV);
      const f32x2 me = both(state8::pow2(141 - mb)), ve = both(state8::pow2(156 - vb)), up = both(state8::pow2(127 + 120));
      uint32_t zero = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t c[4];
        unsigned short half[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int j = 4 * k + 2 * q;
          const uint32_t h0 = state8::mix_folded(key ^ (uint32_t)j), h1 = state8::mix_folded(key ^ (uint32_t)(j + 1));
          float y0, y1;
          unpack2(mul2(pack2(m[j], m[j + 1]), me), y0, y1);
          y0 = __uint_as_float((__float_as_uint(y0) + state8::random_m(h0)) & 0xfff00000u);
          y1 = __uint_as_float((__float_as_uint(y1) + state8::random_m(h1)) & 0xfff00000u);
          unpack2(mul2(pack2(y0, y1), up), y0, y1);
          asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(half[q]) : "f"(y1), "f"(y0));
          unpack2(mul2(pack2(v[j], v[j + 1]), ve), y0, y1);
          // (bits + random) << 4; the four bits more of the hash lie below all others and carry nothing
          c[2 * q] = (__float_as_uint(y0) << 4) + (h0 >> 8);
          c[2 * q + 1] = (__float_as_uint(y1) << 4) + (h1 >> 8);
        }
        reinterpret_cast<uint32_t*>(mq)[k] = (uint32_t)half[0] | (uint32_t)half[1] << 16;
        const uint32_t vw = __byte_perm(__byte_perm(c[0], c[1], 0x0073), __byte_perm(c[2], c[3], 0x0073), 0x5410);
        zero |= (vw - 0x01010101u) & ~vw;
        reinterpret_cast<uint32_t*>(vq)[k] = vw;
      }
      if (zero & 0x80808080u) {  // some code is 0
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          uint32_t& vw = reinterpret_cast<uint32_t*>(vq)[j / 4];
          if (v[j] > 0.f && (vw >> (8 * (j & 3)) & 0xffu) == 0) vw |= 1u << (8 * (j & 3));
        }
      }
    } else {
      mt = vt = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        // an element that is not finite does not set the block's exponent
        const uint32_t a = __float_as_uint(m[j]) & 0x7fffffffu, b = __float_as_uint(v[j]) & 0x7fffffffu;
        if (a < 0x7f800000u) mt = max(mt, a);
        if (b < 0x7f800000u) vt = max(vt, b);
      }
      const unsigned pair = 3u << (threadIdx.x & 30);
      mt = max(mt, __shfl_xor_sync(pair, mt, 1));
      vt = max(vt, __shfl_xor_sync(pair, vt, 1));
      mb = state8::block_exp(mt, state8::kMinExpM);
      vb = state8::block_exp(vt, state8::kMinExpV);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t r = state8::mix_folded(key ^ (uint32_t)j);
        mq[j] = state8::encode_m(m[j], mb, state8::random_m(r));
        vq[j] = state8::encode_v(v[j], vb, state8::random_v(r));
      }
    }
    if (at < coded) {
      *reinterpret_cast<uint4*>(mc + at) = *reinterpret_cast<uint4*>(mq);
      *reinterpret_cast<uint4*>(vc + at) = *reinterpret_cast<uint4*>(vq);
      if ((threadIdx.x & 1) == 0) {
        ms[at >> 5] = (uint8_t)mb;
        vs[at >> 5] = (uint8_t)vb;
      }
    }
    if (!vec) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const unsigned i = j * kThreads + threadIdx.x;
        if (start + i < len) {
          const float y = s_w[padded(i)];
          p[start + i] = from_f<P>(y);
          if (kMaster) w[start + i] = y;
        }
      }
      __syncthreads();  // the next part may be staged too
    }
  }
}

// ---------------------------------------------------------------- 8-bit states to values and back
// Bound by HBM: 67 M codes to bf16 33 us (6.1 TB/s); 16 codes per thread with 16-byte stores took 40.
// A block of 32 codes per thread (`vec`: the addresses allow accesses of 32 bytes), else one by one.
template <typename T, int kMoment>
__global__ void __launch_bounds__(kThreads)
adamw8_values_kernel(const uint8_t* codes, const uint8_t* exps, long long n, int vec, T* out) {
  const long long at = ((long long)blockIdx.x * kThreads + threadIdx.x) * 32;
  if (at >= n) return;
  const int b = exps[at >> 5];
  if (vec && at + 32 <= n) {
    alignas(32) uint8_t c[32];
    load_vec(codes + at, c);
    const f32x2 factor = both(kMoment == 1 ? state8::factor_m(b) : state8::factor_v(b));
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 16 at a time: fewer registers
      alignas(32) T x[16];
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(c)[(16 * h + j) / 4];
        float lo, hi;
        unpack2(mul2(kMoment == 1 ? decode_m2(w, j & 2) : decode_v2(w, j & 2), factor), lo, hi);
        x[j] = from_f<T>(lo);
        x[j + 1] = from_f<T>(hi);
      }
      store_vec(out + at + 16 * h, x);
    }
    return;
  }
  for (int j = 0; j < 32 && at + j < n; ++j) {
    const uint8_t c = codes[at + j];
    out[at + j] = from_f<T>(kMoment == 1 ? state8::decode_m(c, b)
                                         : state8::decode_v(c >= state8::kInfiniteV ? (uint8_t)255 : c, b));
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

// The lists of a group that name memory: where each tensor lies and how many bytes it has there.
template <typename Visit>
void for_lists(const fm_adamw_group& g, Visit visit) {
  const bool eight = g.state_bits == 8;
  const auto list = [&](const auto* at, bool written, auto bytes) {
    visit(g.count, written, [=, &g](int i) -> Range {
      const size_t n = (size_t)g.numels[i];
      const uintptr_t begin = (uintptr_t)at[i];
      return {begin, begin + bytes(n), written};
    });
  };
  const auto each = [](size_t unit) { return [unit](size_t n) { return n * unit; }; };
  const auto codes = [](size_t n) { return (n + 31) / 32 * 32; };
  const auto scales = [](size_t n) { return (n + 31) / 32; };
  list(g.params, true, each(dtype_bytes(g.p_dtype)));
  list(g.grads, false, each(dtype_bytes(g.g_dtype)));
  for (void* const* moments : {g.exp_avg, g.exp_avg_sq})
    if (eight) list(moments, true, codes);
    else list(moments, true, each(4));
  if (g.masters) list(g.masters, true, each(4));
  if (eight) {
    list(g.exp_avg_scale, true, scales);
    list(g.exp_avg_sq_scale, true, scales);
  }
  list(g.steps, true, [](size_t) { return (size_t)4; });
  if (g.lr_device) visit(1, false, [&](int) -> Range { return {(uintptr_t)g.lr_device, (uintptr_t)g.lr_device + 4, false}; });
}

// Refuses a call whose written memory overlaps anything else of the call: two threads would race.
// Where the lists are in the order of their addresses and lie apart from one another, neighbours are all there is to
// compare; else all of it is sorted.
int check_ranges(const fm_adamw_group* groups, int ngroups, const float* scale) {
  const auto less = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  std::vector<Range> hulls;
  hulls.reserve(ngroups * 9 + 1);
  bool apart = true;
  size_t total = 1;
  for (int gi = 0; gi < ngroups; ++gi) {
    if (groups[gi].count == 0) continue;
    for_lists(groups[gi], [&](int count, bool written, auto at) {
      total += count;
      Range hull = {0, 0, written};
      for (int i = 0; i < count && apart; ++i) {
        const Range x = at(i);
        if (x.begin == x.end) continue;
        if (hull.end == 0) hull.begin = x.begin;
        apart = x.begin >= hull.end;
        hull.end = x.end;
      }
      if (hull.end != 0) hulls.push_back(hull);
    });
  }
  if (scale) hulls.push_back({(uintptr_t)scale, (uintptr_t)scale + 4, false});
  if (apart) {
    std::sort(hulls.begin(), hulls.end(), less);
    for (size_t i = 1; i < hulls.size(); ++i) apart = apart && hulls[i - 1].end <= hulls[i].begin;
    if (apart) return FM_OK;
  }
  std::vector<Range> r;
  r.reserve(total);
  if (scale) r.push_back({(uintptr_t)scale, (uintptr_t)scale + 4, false});
  std::vector<size_t> runs = {0, r.size()};  // where the sorted lists begin, and the end
  for (int gi = 0; gi < ngroups; ++gi) {
    if (groups[gi].count == 0) continue;
    for_lists(groups[gi], [&](int count, bool, auto at) {
      const size_t from = r.size();
      for (int i = 0; i < count; ++i) {
        const Range x = at(i);
        if (x.begin != x.end) r.push_back(x);
      }
      if (!std::is_sorted(r.begin() + from, r.end(), less)) std::sort(r.begin() + from, r.end(), less);
      runs.push_back(r.size());
    });
  }
  for (size_t step = 1; step + 1 < runs.size(); step *= 2)  // runs[i] .. runs[i + step] is in order
    for (size_t i = 0; i + step + 1 < runs.size(); i += 2 * step)
      std::inplace_merge(r.begin() + runs[i], r.begin() + runs[i + step],
                         r.begin() + runs[std::min(i + 2 * step, runs.size() - 1)], less);
  uintptr_t any = 0, written = 0;
  for (const Range& x : r) {
    if (x.begin < (x.written ? any : written)) return fail(FM_ERR_INVALID, "tensors of the step overlap (the same parameter twice?)");
    any = std::max(any, x.end);
    if (x.written) written = std::max(written, x.end);
  }
  return FM_OK;
}

int check_group(const fm_adamw_group& g, int gi) {
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
  const size_t pb = dtype_bytes(g.p_dtype), gb = dtype_bytes(g.g_dtype);
  for (int i = 0; i < g.count; ++i) {
    const int64_t n = g.numels[i];
    if (n < 0 || n > (int64_t)1 << 38) return fail(FM_ERR_INVALID, "group %d: bad element count at %d", gi, i);
    if (!g.steps[i] || !aligned(g.steps[i], 4)) return fail(FM_ERR_INVALID, "group %d: bad step count at %d", gi, i);
    if (n == 0) continue;
    if (!g.params[i] || !g.grads[i] || !g.exp_avg[i] || !g.exp_avg_sq[i] || (g.masters && !g.masters[i]))
      return fail(FM_ERR_INVALID, "group %d: null tensor pointer at %d", gi, i);
    if (!aligned(g.params[i], pb) || !aligned(g.grads[i], gb) || (g.masters && !aligned(g.masters[i], 4)) ||
        !aligned(g.exp_avg[i], g.state_bits == 8 ? 16 : 4) || !aligned(g.exp_avg_sq[i], g.state_bits == 8 ? 16 : 4))
      return fail(FM_ERR_INVALID, "group %d: misaligned tensor at %d", gi, i);
    if (g.state_bits == 8 && (!g.exp_avg_scale[i] || !g.exp_avg_sq_scale[i]))
      return fail(FM_ERR_INVALID, "group %d: null scales at %d", gi, i);
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tab.first[tab.count]);
  cfg.blockDim = dim3(tab.threads);
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
  if (tab.whole) return launch_table<adamw_kernel<P, G, kMaster, true, N>>(tab, dependent, stream);
  return launch_table<adamw_kernel<P, G, kMaster, false, N>>(tab, dependent, stream);
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

  template <int N>
  int launch_part() {
    Table<N> t;
    std::copy(tab.e, tab.e + tab.count, t.e);
    std::copy(tab.first, tab.first + tab.count + 1, t.first);
    std::copy(tab.h, tab.h + hypers, t.h);
    t.scale = tab.scale;
    t.count = tab.count;
    t.parts = tab.parts;
    t.threads = tab.threads;
    t.whole = tab.whole;
    return launch(t, kind, dependent, stream);
  }

  int flush() {
    if (tab.count == 0) return FM_OK;
    int rc;
    if (tab.count <= kSmallTable) rc = launch_part<kSmallTable>();
    else if (tab.count <= kMediumTable) rc = launch_part<kMediumTable>();
    else rc = launch(tab, kind, dependent, stream);
    tab.count = 0;
    hypers = 0;
    last_group = -1;
    dependent = false;
    return rc;
  }

  int add(const fm_adamw_group& g, int gi, int i) {
    const int64_t n = g.numels[i];
    const int tile = g.state_bits == 8 ? tab.parts * kPart8 : tab.threads * kEach32;
    const int64_t tiles = (n + tile - 1) / tile;
    if (tab.count > 0 && (tab.count == kLargeTable || (last_group != gi && hypers == kMaxHyper) ||
                          tab.first[tab.count] + tiles > 0x7fffffffLL)) {
      const int rc = flush();
      if (rc != FM_OK) return rc;
    }
    if (tab.count == 0) tab.first[0] = 0;
    if (last_group != gi) {
      Hyper& h = tab.h[hypers++];
      h.lr = g.lr; h.beta1 = g.beta1; h.beta2 = g.beta2; h.lr_dev = g.lr_device;
      h.wd = g.weight_decay;
      h.b1 = (float)g.beta1; h.omb1 = (float)(1.0 - g.beta1);
      h.b2 = (float)g.beta2; h.omb2 = (float)(1.0 - g.beta2);
      h.root_omb2 = (float)std::sqrt(1.0 - g.beta2);
      // 8 bits: the smallest stored second moment is 2^-126; a step may leave less, whose approximate root is 0.
      // 32 bits: eps sqrt(1 - b2^t) >= eps sqrt(1 - b2) stays a normal number, or the approximate reciprocal
      // were infinite where there never was a gradient.
      const float least = g.state_bits == 8 ? 0x1p-64f : g.eps > 0.0 ? 0x1p-125f / h.root_omb2 : 0.f;
      h.eps = std::max((float)g.eps, least);
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
    const size_t wide = g.state_bits == 8 ? 16 : 32;  // of the moments
    e.vec = aligned(e.p, 32) && aligned(e.g, 32) && aligned(e.w, 32) && aligned(e.m, wide) && aligned(e.v, wide);
    tab.first[tab.count + 1] = tab.first[tab.count] + (unsigned)tiles;
    ++tab.count;
    return FM_OK;
  }
};

// Parts of a tile with 8-bit states: what a block spends on its tensor's coefficients is shared by up to
// 8 of them, as many as leave every SM 12 blocks (5 or 6 are resident).  67 M bf16 elements, at an earlier
// step of the kernel: 1 part 137 us, 2 132, 4 130, 8 129, 16 no better.
// A tile's random numbers take their upper index bits from its first element, so no tile may hold indices on both
// sides of a multiple of 2^32: where there are that many elements tiles have 8 parts, which divide it.
constexpr long long kBlocksPerSm = 12, kMostSms = 1024;
static_assert((1LL << 32) % (kMaxParts * kPart8) == 0);
static_assert((1LL << 32) / (kPart8 * kBlocksPerSm * kMostSms + 1) >= kMaxParts);
int parts_of(long long elements) {
  const long long parts = elements / (kPart8 * kBlocksPerSm * std::min<long long>(sm_count(), kMostSms) + 1);
  return parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : (int)parts;
}

// The counts of what is added, advanced by as many launches as that takes.
struct Counts {
  CountTable tab;
  cudaStream_t stream;
  bool launched = false;
  int add(float* step) {
    tab.step[tab.count++] = step;
    return tab.count == kCountTable ? flush() : FM_OK;
  }
  int flush() {
    if (tab.count == 0) return FM_OK;
    adamw_count_kernel<<<1, kThreads, 0, stream>>>(tab);
    tab.count = 0;
    launched = true;
    FM_CUDA_CHECK(cudaGetLastError());
    return FM_OK;
  }
};

int adamw_step(const fm_adamw_group* groups, int ngroups, const float* scale, cudaStream_t stream) {
  size_t tensors = 0;
  for (int gi = 0; gi < ngroups; ++gi) {
    const int rc = check_group(groups[gi], gi);
    if (rc != FM_OK) return rc;
    tensors += groups[gi].count;
  }
  if (tensors == 0) return FM_OK;
  if (!aligned(scale, 4)) return fail(FM_ERR_INVALID, "misaligned gradient scale");
  int rc = check_ranges(groups, ngroups, scale);
  if (rc != FM_OK) return rc;

  // the kinds of the call, their elements and largest tensors
  struct Work {
    Kind kind;
    long long elements = 0, largest = 0;
  };
  std::vector<Work> works;
  std::vector<int> work_of(ngroups, 0);
  for (int gi = 0; gi < ngroups; ++gi) {
    const Kind k = kind_of(groups[gi]);
    size_t w = 0;
    while (w < works.size() && !(works[w].kind == k)) ++w;
    if (w == works.size()) works.push_back({k});
    work_of[gi] = (int)w;
    for (int i = 0; i < groups[gi].count; ++i) {
      works[w].elements += groups[gi].numels[i];
      works[w].largest = std::max(works[w].largest, (long long)groups[gi].numels[i]);
    }
  }
  // One block per tensor saves the launch of the counts, 2 us of host time.  On the device that is 3.7 us
  // instead of 4.1 for 65 tensors of 1000 f32 elements and 4.3 either way for 65 of 4096, but 6.1 instead of
  // 5.3 for 65 of 8192 (8-bit states 4.0 / 4.8, 4.5 / 4.3, 6.3 / 4.8): up to 4096 elements.
  const auto whole = [&](const Work& w) {
    return w.largest <= (w.kind.bits == 8 ? kWholeParts * kPart8 : kMaxThreads * kEach32);
  };
  Counts counts;
  counts.tab.count = 0;
  counts.tab.scale = scale;
  counts.stream = stream;
  for (int gi = 0; gi < ngroups; ++gi) {
    const bool all = !whole(works[work_of[gi]]);
    for (int i = 0; i < groups[gi].count && rc == FM_OK; ++i)
      if (all || groups[gi].numels[i] == 0) rc = counts.add(groups[gi].steps[i]);
  }
  if (rc == FM_OK) rc = counts.flush();
  if (rc != FM_OK) return rc;

  Batch batch;
  batch.tab.count = 0;
  batch.tab.scale = scale;
  batch.stream = stream;
  batch.dependent = counts.launched && options().pdl != 0;
  for (const bool now : {false, true}) {  // what waits for the counts follows them directly
    for (size_t w = 0; w < works.size(); ++w) {
      const Work& work = works[w];
      if (whole(work) != now || work.elements == 0) continue;
      batch.kind = work.kind;
      batch.tab.whole = now;
      batch.tab.threads = kThreads;
      batch.tab.parts = parts_of(work.elements);
      if (now) {
        batch.tab.parts = (int)((work.largest + kPart8 - 1) / kPart8);
        while (work.kind.bits == 32 && batch.tab.threads * kEach32 < work.largest) batch.tab.threads *= 2;
      }
      for (int gi = 0; gi < ngroups; ++gi) {
        if (work_of[gi] != (int)w) continue;
        for (int i = 0; i < groups[gi].count; ++i) {
          if (groups[gi].numels[i] == 0) continue;
          rc = batch.add(groups[gi], gi, i);
          if (rc != FM_OK) return rc;
        }
      }
      rc = batch.flush();
      if (rc != FM_OK) return rc;
    }
  }
  return FM_OK;
}

int simple_grid(long long n) {
  const long long want = (n + kThreads - 1) / kThreads, most = (long long)sm_count() * 8;
  return (int)(want < most ? want : most);
}

int check_moment(const void* a, const void* b, const void* c, int64_t n, int moment) {
  if (n < 0 || n > (int64_t)1 << 38) return fail(FM_ERR_INVALID, "bad element count");
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
  if (!aligned(out, dtype_bytes(out_dtype))) return fail(FM_ERR_INVALID, "misaligned values");
  if (n == 0) return FM_OK;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int vec = aligned(codes, 32) && aligned(out, 32);
  const unsigned grid = (unsigned)((n + kThreads * 32 - 1) / (kThreads * 32));
  auto go = [&](auto* o) {
    using T = std::remove_pointer_t<decltype(o)>;
    if (moment == 1) adamw8_values_kernel<T, 1><<<grid, kThreads, 0, st>>>(c, s, n, vec, o);
    else adamw8_values_kernel<T, 2><<<grid, kThreads, 0, st>>>(c, s, n, vec, o);
  };
  if (out_dtype == FM_F32) go(static_cast<float*>(out));
  else if (out_dtype == FM_BF16) go(static_cast<__nv_bfloat16*>(out));
  else go(static_cast<__half*>(out));
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
  if (!aligned(values, dtype_bytes(v_dtype))) return fail(FM_ERR_INVALID, "misaligned values");
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
