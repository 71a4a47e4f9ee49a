// Driver of the data-race check (see race_check.cpp) for the norms' gradients where a workgroup goes from row to row: more than 512 rows
// (2048 of up to 512 columns), in every form of a row. Results are not checked here; the exit status is the sanitizer's.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "../../include/moe_gg.h"

static uint32_t rng_state = 4242u;
static uint32_t rnd() { rng_state = rng_state * 1664525u + 1013904223u; return rng_state >> 8; }
static std::vector<uint16_t> halves(size_t n) {  // -2 .. 2 in either 16-bit type's patterns
  static const uint16_t code[5] = {0xC000, 0xBC00, 0x0000, 0x3C00, 0x4000};
  std::vector<uint16_t> v(n + 64);
  for (auto& x : v) x = code[rnd() % 5];
  return v;
}
static int failures = 0;

static void norms(int T, int d, int kind, bool post, bool with_y) {
  const int dtype = MOE_GG_DTYPE_BF16;
  auto y = halves((size_t)T * d), h = halves((size_t)T * d), gz = halves((size_t)T * d), gh = halves((size_t)T * d);
  auto wp = halves(d), wn = halves(d), g = halves(T > d ? T : d);
  auto gy = y, gr = h, g1 = wp, g2 = wn, g3 = g;
  const size_t n = moe_gg_block_norm_backward_workspace(T, d);
  std::vector<char> w(n + 512);
  void* work = (void*)(((uintptr_t)w.data() + 255) & ~(uintptr_t)255);
  post = post && with_y;
  kind = with_y ? kind : 0;
  const int rc = moe_gg_block_norm_backward(gh.data(), d, gz.data(), d, with_y ? y.data() : nullptr, d, h.data(), d, post ? wp.data() : nullptr,
                                            kind ? g.data() : nullptr, kind, wn.data(), 1.f, 0.5f, 1e-6f, with_y ? gy.data() : nullptr, gr.data(),
                                            post ? g1.data() : nullptr, kind ? g3.data() : nullptr, g2.data(), T, d, dtype, dtype, dtype, work, n, nullptr);
  std::printf("block_norm_backward T %5d d %5d gate %d %s rc %d\n", T, d, kind, with_y ? "" : "norm alone", rc);
  std::fflush(stdout);
  if (rc != 0) ++failures;
}

int main() {
  norms(2100, 16, 2, true, true);
  norms(516, 520, 1, true, true);
  norms(516, 600, 0, true, false);
  norms(516, 2056, 2, true, true);
  norms(516, 4104, 1, true, true);
  norms(514, 8200, 2, true, true);
  std::printf("calls that returned an error: %d\n", failures);
  return failures ? 1 : 0;
}
