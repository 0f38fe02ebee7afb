// Arithmetic of optimizer states held in 8 bits, as host-compilable code (tests run it on the CPU).
//
// A tensor's moment is stored in blocks of 32 consecutive elements: one byte per element and one
// exponent byte b per block, the biased fp32 exponent of the block's largest finite magnitude.  In
// units of 2^(b - 127) the largest element of a block lies in [1, 2).
//   first moment:   sign | e4m3.  A fp32 number scaled by 2^-113 has, in [0, 2), a biased exponent
//                   of at most 14, and the seven bits above bit 20 of its pattern ARE the code:
//                   e4m3 with its subnormals, because fp32 goes subnormal at the same place.  127
//                   stands for "not a number".
//   second moment:  e5m3 without a sign, the same way with 2^-98.  255 stands for infinity, and a
//                   positive value never becomes 0 (a zero under the root would turn any momentum
//                   into a huge update).
// The second moment gets its fifth exponent bit because it is a square: within a block it spans
// twice the binades of the gradient (2^-31 of the largest element here, 2^-15 in the gradient).
//
// Rounding adds a random number of 20 bits below the code's last bit and cuts: up with the chance
// of the distance to the code below, so the stored value is right on average.  Rounding to nearest
// would freeze the moments: a step moves v by (1 - beta2) (g^2 - v), a thousandth of it at
// beta2 = 0.999, while half a step of the code is 3 to 6 % of the value.
#pragma once
#include <cstdint>
#include <cstring>

#ifdef __CUDACC__
#define FM_HD __host__ __device__ __forceinline__
#else
#define FM_HD inline
#endif

namespace fm {
namespace state8 {

constexpr int kBlock = 32;
// Range of the exponent byte: from 17 and 32 on the smallest code of a block is a normal fp32 number.
constexpr int kMinExpM = 17, kMinExpV = 32, kMaxExp = 253;
// Second-moment codes from here on are only written where they stand for infinity (a largest element beyond 2^126
// leaves the binade of its exponent byte); the kernels, which read codes as f16 bits, take them all for it.
constexpr int kInfiniteV = 248;
constexpr uint32_t kNearest = 1u << 19;                   // the "random" number of rounding to nearest

FM_HD uint32_t bits_of(float x) {
#ifdef __CUDA_ARCH__
  return __float_as_uint(x);
#else
  uint32_t u;
  std::memcpy(&u, &x, 4);
  return u;
#endif
}
FM_HD float float_of(uint32_t u) {
#ifdef __CUDA_ARCH__
  return __uint_as_float(u);
#else
  float x;
  std::memcpy(&x, &u, 4);
  return x;
#endif
}
// 2^(e - 127) for 1 <= e <= 254
FM_HD float pow2(int e) { return float_of((uint32_t)e << 23); }

// A bijection of 32 bits in the published shape of integer finalizers (Appleby, 2008: xor-shift, odd factor,
// xor-shift, odd factor, xor-shift).  The factors are this file's own, found by a search for even avalanche: over
// 2^22 inputs flipping any input bit flips any output bit with a chance of 0.497 to 0.503.
FM_HD uint32_t mix_folded(uint32_t x) {  // behind the first xor-shift
  x *= 0xa1c7d3e7u;
  x ^= x >> 15;
  x *= 0x2e3ad36du;
  return x ^ (x >> 16);
}
FM_HD uint32_t mix(uint32_t x) { return mix_folded(x ^ (x >> 16)); }
// Key of a tensor's step: `count` is the step's number, counted from 1.
FM_HD uint32_t step_key(uint32_t seed, uint32_t count) { return mix(mix(seed) + count); }
// Key of the elements whose index has `hi` above bit 32.
FM_HD uint32_t index_key(uint32_t key, uint32_t hi) { return mix(key + hi); }
// 32 random bits of the element with the low index bits `lo`; the first moment takes the lower 20,
// the second the upper 20.  They share 8 bits, the first's highest and the second's lowest.
FM_HD uint32_t random_bits(uint32_t key_hi, uint32_t lo) { return mix(lo ^ key_hi); }
FM_HD uint32_t random_m(uint32_t h) { return h & 0xfffffu; }
FM_HD uint32_t random_v(uint32_t h) { return h >> 12; }

// Exponent byte of a block from the bit pattern of its largest finite magnitude.
FM_HD int block_exp(uint32_t max_bits, int lowest) {
  int e = (int)(max_bits >> 23);
  e = e < lowest ? lowest : e;
  return e > kMaxExp ? kMaxExp : e;
}

FM_HD uint8_t encode_m(float x, int b, uint32_t r) {
  const uint32_t sign = (bits_of(x) >> 24) & 0x80u, mag = bits_of(x) & 0x7fffffffu;
  if (mag >= 0x7f800000u) return (uint8_t)(sign | 127u);
  // two factors: 2^(14 - b) alone leaves the range of fp32
  const float w = float_of(mag) * pow2(254 - b) * pow2(14);
  const uint32_t c = (bits_of(w) + r) >> 20;
  return (uint8_t)(sign | (c > 126u ? 126u : c));
}
FM_HD uint8_t encode_v(float x, int b, uint32_t r) {
  const uint32_t mag = bits_of(x) & 0x7fffffffu;
  if (mag >= 0x7f800000u) return 255;
  const float w = float_of(mag) * pow2(254 - b) * pow2(29);
  const uint32_t c = (bits_of(w) + r) >> 20;
  if (c == 0) return mag != 0 ? 1 : 0;
  return (uint8_t)(c > 254u ? 254u : c);
}
// Factors of a block's codes read as numbers with the exponent offsets 7 (e4m3) and 15 (e5m3): 2^(b - 134)
// and 2^(b - 141).  An exponent byte below the smallest counts as the smallest.
FM_HD float factor_m(int b) { return pow2((b > kMinExpM ? b : kMinExpM) - 7); }
FM_HD float factor_v(int b) { return pow2((b > kMinExpV ? b : kMinExpV) - 14); }
FM_HD float decode_m(uint8_t c, int b) {
  const uint32_t mag = c & 127u;
  if (mag == 127u) return float_of(0x7fc00000u);
  const float x = float_of(mag << 20) * pow2(247) * factor_m(b);
  return (c & 128u) ? -x : x;
}
FM_HD float decode_v(uint8_t c, int b) {
  if (c == 255u) return float_of(0x7f800000u);
  return float_of((uint32_t)c << 20) * pow2(239) * factor_v(b);
}

}  // namespace state8
}  // namespace fm
