// Host check: what a code of an 8-bit optimizer state stands for at every exponent byte, those below the
// smallest that is written among them (csrc/state8.cuh).
#include <cmath>
#include <cstdio>

#include "state8.cuh"

using namespace fm::state8;

// value of a code without sign at exponent byte b: `first` is the exponent of the smallest normal code
static double value(int c, int b, int lowest, int first) {
  const int e = c >> 3, f = c & 7;
  b = b < lowest ? lowest : b;
  return e == 0 ? std::ldexp(f, b - 127 + first - 3) : std::ldexp(8 + f, b - 127 + first - 4 + e);
}

int main() {
  int fails = 0;
  for (int b = 0; b < 256; ++b) {
    for (int c = 0; c < 127; ++c) {
      const float x = (float)value(c, b, kMinExpM, -13);
      fails += decode_m((uint8_t)c, b) != x || decode_m((uint8_t)(c | 128), b) != -x;
    }
    for (int c = 0; c < 255; ++c) fails += decode_v((uint8_t)c, b) != (float)value(c, b, kMinExpV, -28);
    fails += !std::isnan(decode_m(127, b)) || !std::isnan(decode_m(255, b)) || !std::isinf(decode_v(255, b));
  }
  // the unit of the exponent byte: code 112 of the first moment and code 232 of the second
  fails += decode_m(112, 127) != 1.f || decode_v(232, 127) != 1.f;
  if (fails) std::fprintf(stderr, "%d failures\n", fails);
  else std::printf("OK\n");
  return fails != 0;
}
