// exp_neg_p against the C library's exp on both sides of 0, up to f64's end:
// at most 2 ulp apart.  Prints "<failures> <cases>".
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "../metallix_amd/csrc/mxs_math.h"

int main(void) {
  uint64_t state = 0x2545f4914f6cdd1dull;
  long fail = 0, cases = 0;
  auto one = [&](double x) {
    const double a = exp(x), b = mxs::exp_neg_p(x);
    int64_t p, q;
    memcpy(&p, &a, 8);
    memcpy(&q, &b, 8);
    ++cases;
    if (p - q > 2 || q - p > 2) ++fail;
  };
  for (int i = 0; i < 4000000; ++i) {
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    const double u = (double)(state >> 11) * 0x1.0p-53;
    one(i % 2 ? 709.0 * u : i % 4 ? u : 1e-6 * u);
  }
  const double edge[] = {0.0, 0.35, 0.34657359027997264, 0.34657359027997270, 600.0, 600.5, 640.0, 708.9, 709.0};
  for (double x : edge) one(x);
  printf("%ld %ld\n", fail, cases);
  return 0;
}
