// Host check of the arithmetic of 8-bit optimizer states (csrc/state8.cuh), without a GPU: every code
// of every exponent byte, the rounding of whole grids of values, and values that are not finite.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include <limits>

#include "state8.cuh"

using namespace fm::state8;

static int fails = 0;
#define CHECK(cond, ...)                                     \
  do {                                                       \
    if (!(cond) && ++fails <= 20) {                          \
      std::fprintf(stderr, "line %d: %s: ", __LINE__, #cond); \
      std::fprintf(stderr, __VA_ARGS__);                     \
      std::fprintf(stderr, "\n");                            \
    }                                                        \
  } while (0)

// value of a code at exponent byte b, from the definition
static double value_m(int c, int b) {
  const int e = (c & 127) >> 3, f = c & 7;
  const double x = e == 0 ? std::ldexp(f, b - 127 - 16) : std::ldexp(8 + f, b - 127 - 17 + e);
  return c & 128 ? -x : x;
}
static double value_v(int c, int b) {
  const int e = c >> 3, f = c & 7;
  return e == 0 ? std::ldexp(f, b - 127 - 31) : std::ldexp(8 + f, b - 127 - 32 + e);
}

int main() {
  long checked = 0;
  const float inf = std::numeric_limits<float>::infinity(), nan = std::numeric_limits<float>::quiet_NaN();
  // 1. decode is the definition (where fp32 holds it) and encode to nearest, or with any random
  //    number, gives the code back
  for (int b = kMinExpM; b <= kMaxExp; ++b)
    for (int c = 0; c < 256; ++c) {
      if ((c & 127) == 127) { CHECK(std::isnan(decode_m((uint8_t)c, b)), "c %d b %d", c, b); continue; }
      const float x = decode_m((uint8_t)c, b);
      CHECK(x == (float)value_m(c, b), "c %d b %d", c, b);
      if (!std::isfinite(x)) continue;
      const uint32_t rs[] = {0u, 1u, kNearest, 0xfffffu};
      for (uint32_t r : rs) CHECK(encode_m(x, b, r) == c, "c %d b %d r %u got %d", c, b, r, encode_m(x, b, r));
      ++checked;
    }
  for (int b = kMinExpV; b <= kMaxExp; ++b)
    for (int c = 0; c < 256; ++c) {
      if (c == 255) { CHECK(std::isinf(decode_v(255, b)), "b %d", b); continue; }
      const float x = decode_v((uint8_t)c, b);
      CHECK(x == (float)value_v(c, b), "c %d b %d", c, b);
      if (!std::isfinite(x)) continue;
      const uint32_t rs[] = {0u, 1u, kNearest, 0xfffffu};
      for (uint32_t r : rs) CHECK(encode_v(x, b, r) == c, "c %d b %d r %u got %d", c, b, r, encode_v(x, b, r));
      ++checked;
    }
  // 2. between two neighbouring codes exactly the share of the random numbers that the distance asks
  //    for goes up: at x = low + k/64 of a step, r goes up iff k/64 + r/2^20 >= 1
  for (int moment = 1; moment <= 2; ++moment)
    for (int b : {moment == 1 ? kMinExpM : 40, 60, 127, 200})
      for (int c = 0; c < (moment == 1 ? 120 : 240); ++c) {
        const double lo = moment == 1 ? value_m(c, b) : value_v(c, b), hi = moment == 1 ? value_m(c + 1, b) : value_v(c + 1, b);
        if (hi < std::ldexp(1.0, -120)) continue;
        for (int k = 0; k < 64; ++k) {
          const float x = (float)(lo + (hi - lo) * k / 64);
          const uint32_t edge = (1u << 20) - (uint32_t)k * (1u << 14);  // first r that goes up
          for (int d = -1; d <= 1; ++d) {
            const int64_t r = (int64_t)edge + d;
            if (r < 0 || r >= (1 << 20)) continue;
            int want = c + (d >= 0);
            if (moment == 2 && want == 0 && x > 0) want = 1;
            const int got = moment == 1 ? encode_m(x, b, (uint32_t)r) : encode_v(x, b, (uint32_t)r);
            CHECK(got == want, "moment %d b %d c %d k %d d %d: %d", moment, b, c, k, d, got);
            if (moment == 1) CHECK(encode_m(-x, b, (uint32_t)r) == (want | 128), "negative, b %d c %d k %d", b, c, k);
            ++checked;
          }
        }
      }
  // 3. the largest element of a block: any magnitude, its own exponent byte, never saturates
  for (uint32_t u = 1; u < 0x7f800000u; u += 0x10001u) {
    const float x = float_of(u);
    const int bm = block_exp(u, kMinExpM), bv = block_exp(u, kMinExpV);
    CHECK(bm >= kMinExpM && bm <= kMaxExp && bv >= kMinExpV && bv <= kMaxExp, "u %08x", u);
    for (uint32_t r : {0u, 0xfffffu}) {
      const int cm = encode_m(x, bm, r), cv = encode_v(x, bv, r);
      CHECK((cm & 127) <= 126 && cv <= 254 && cv >= 1, "u %08x codes %d %d", u, cm, cv);
      if (u >= 0x10000000u && u < 0x7f000000u) {  // block maximum in the binade that b names
        CHECK(cm >= 112 && cm <= 120, "u %08x code %d", u, cm);
        CHECK(cv >= 232 && cv <= 240, "u %08x code %d", u, cv);
        CHECK(std::fabs(decode_m((uint8_t)cm, bm) / x - 1) <= 0.125, "u %08x", u);
        CHECK(std::fabs(decode_v((uint8_t)cv, bv) / x - 1) <= 0.125, "u %08x", u);
      }
      ++checked;
    }
  }
  // 4. values that are not finite
  for (int b : {17, 127, 253}) {
    CHECK((encode_m(nan, b, 0) & 127) == 127 && (encode_m(inf, b, 0) & 127) == 127 && (encode_m(-inf, b, 0) & 127) == 127, "b %d", b);
    CHECK(encode_v(nan, b, 0) == 255 && encode_v(inf, b, 0) == 255, "b %d", b);
    CHECK(encode_m(0.f, b, 0xfffffu) == 0 && encode_v(0.f, b, 0xfffffu) == 0, "b %d", b);
  }
  // 5. random bits: the share that goes up, over elements, steps and seeds, is the distance asked for.
  //    N = 2^20 draws of a chance p: standard deviation below 1/2^11; five of them
  const int kDraws = 1 << 20;
  for (int way = 0; way < 3; ++way) {
    long up_m[3] = {0, 0, 0}, up_v[3] = {0, 0, 0};
    const uint32_t edge[3] = {1u << 18, 1u << 19, 1000000u};
    for (int i = 0; i < kDraws; ++i) {
      const uint32_t seed = way == 2 ? i : 7, step = way == 1 ? i + 1 : 3, lo = way == 0 ? i : 12345;
      const uint32_t h = random_bits(index_key(step_key(seed, step), 0), lo);
      for (int k = 0; k < 3; ++k) {
        up_m[k] += random_m(h) < edge[k];
        up_v[k] += random_v(h) < edge[k];
      }
    }
    for (int k = 0; k < 3; ++k) {
      const double p = edge[k] / 1048576.0;
      CHECK(std::fabs(up_m[k] / (double)kDraws - p) < 5.0 / 2048, "way %d k %d: %f", way, k, up_m[k] / (double)kDraws);
      CHECK(std::fabs(up_v[k] / (double)kDraws - p) < 5.0 / 2048, "way %d k %d: %f", way, k, up_v[k] / (double)kDraws);
    }
  }
  if (fails) {
    std::fprintf(stderr, "%d failures\n", fails);
    return 1;
  }
  std::printf("OK %ld\n", checked);
  return 0;
}
