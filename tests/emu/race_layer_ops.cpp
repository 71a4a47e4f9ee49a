// Driver of the data-race check (see race_check.cpp) for the adapters, the norms and the gate: every kernel of theirs, with the
// steps of several tiles per workgroup. Results are not checked here; the exit status is the sanitizer's.
#include <cstdint>
#include <cstdio>
#include <vector>

#include "../../include/moe_gg.h"

static uint32_t rng_state = 777u;
static uint32_t rnd() { rng_state = rng_state * 1664525u + 1013904223u; return rng_state >> 8; }
static std::vector<uint16_t> halves(size_t n) {  // -2 .. 2 in either 16-bit type's patterns
  static const uint16_t code[5] = {0xC000, 0xBC00, 0x0000, 0x3C00, 0x4000};
  std::vector<uint16_t> v(n + 64);
  for (auto& x : v) x = code[rnd() % 5];
  return v;
}
static std::vector<float> floats(size_t n) {
  std::vector<float> v(n + 64);
  for (auto& x : v) x = (float)(int)(rnd() % 7) - 3.f;
  return v;
}
static int failures = 0;
static void check(int rc, const char* what) {
  std::printf("%-60s rc %d\n", what, rc);
  std::fflush(stdout);
  if (rc != 0) ++failures;
}
static void* at256(std::vector<char>& v, size_t n) {
  v.assign(n + 512, 0);
  return (void*)(((uintptr_t)v.data() + 255) & ~(uintptr_t)255);
}

static void lora(int T, int K, int N, int R, int L, bool keep, int dtype) {
  std::vector<int32_t> ids(T), perm(T), off(L + 2), scratch(T + L + 1);
  for (int t = 0; t < T; ++t) ids[t] = (int)(rnd() % (L + 1)) - 1;
  check(moe_gg_lora_plan(ids.data(), T, L, perm.data(), off.data(), scratch.data(), nullptr), "lora_plan");
  auto x = halves((size_t)T * K), y = halves((size_t)T * N), a = halves((size_t)L * R * K), b = halves((size_t)L * N * R), out = y, gx = x, ga = a, gb = b;
  auto h = floats((size_t)T * R), s = floats(L);
  std::vector<char> w;
  size_t n = moe_gg_lora_add_workspace(T, L, K, N, R);
  check(moe_gg_lora_add(y.data(), N, x.data(), K, a.data(), b.data(), s.data(), perm.data(), off.data(), L, T, K, N, R, out.data(), N, h.data(), dtype, at256(w, n),
                        n, nullptr), "lora_add");
  n = moe_gg_lora_backward_workspace(T, L, K, N, R, keep);
  check(moe_gg_lora_backward(y.data(), N, x.data(), K, a.data(), b.data(), s.data(), perm.data(), off.data(), L, T, K, N, R, keep ? h.data() : nullptr, x.data(), K,
                             gx.data(), K, ga.data(), gb.data(), dtype, at256(w, n), n, nullptr), "lora_backward");
}

static void norms(int T, int d, int kind, bool post, bool pre, int dtype, int stream, int weights) {
  auto y = halves((size_t)T * d), z = y, gy = y, gz = y;
  std::vector<uint16_t> wp = halves(2 * d), wn = halves(2 * d), g = halves(2 * (T > d ? T : d)), g1 = wp, g2 = wn, g3 = g;
  auto r = floats((size_t)T * d), h = r, gh = r, gr = r;
  check(moe_gg_block_norm(y.data(), d, r.data(), d, post ? wp.data() : nullptr, kind ? g.data() : nullptr, kind, pre ? wn.data() : nullptr, 1.f, 0.5f, 1e-6f, h.data(),
                          pre ? z.data() : nullptr, T, d, dtype, stream, weights, nullptr), "block_norm");
  std::vector<char> w;
  const size_t n = moe_gg_block_norm_backward_workspace(T, d);
  check(moe_gg_block_norm_backward(gh.data(), d, pre ? gz.data() : nullptr, d, y.data(), d, h.data(), d, post ? wp.data() : nullptr, kind ? g.data() : nullptr, kind,
                                   pre ? wn.data() : nullptr, 1.f, 0.5f, 1e-6f, gy.data(), gr.data(), post ? g1.data() : nullptr, kind ? g3.data() : nullptr,
                                   pre ? g2.data() : nullptr, T, d, dtype, stream, weights, at256(w, n), n, nullptr), "block_norm_backward");
  check(moe_gg_block_norm(nullptr, 0, r.data(), d, nullptr, nullptr, 0, wn.data(), 1.f, 1.f, 1e-6f, nullptr, z.data(), T, d, dtype, stream, weights, nullptr), "rms_norm");
}

static void gate(int T, int E, int k, int score, int renorm) {
  auto l = floats((size_t)T * E), w = floats((size_t)T * k), g = l;
  std::vector<int32_t> ids((size_t)T * k);
  check(moe_gg_route_gate(l.data(), MOE_GG_DTYPE_FP32, T, E, k, score, renorm, 1.f, w.data(), ids.data(), nullptr), "route_gate");
  check(moe_gg_route_gate_backward(w.data(), l.data(), MOE_GG_DTYPE_FP32, ids.data(), T, E, k, score, renorm, 1.f, g.data(), nullptr), "route_gate_backward");
}

int main() {
  const int H = MOE_GG_DTYPE_FP16, B = MOE_GG_DTYPE_BF16, F = MOE_GG_DTYPE_FP32;
  lora(9, 72, 80, 16, 3, true, B);         // one kernel
  lora(40, 136, 300, 24, 2, false, H);     // one kernel, two rank blocks; several steps of the gradients
  lora(300, 96, 270, 33, 2, true, H);      // two kernels
  lora(600, 72, 2100, 16, 3, false, B);    // u summed first, several column blocks
  lora(700, 1100, 530, 40, 1, true, B);    // chunks of one adapter
  lora(530, 64, 72, 100, 2, true, B);      // ranks in two rounds
  norms(5, 500, 1, true, true, B, F, B);
  norms(9, 1030, 2, true, true, H, H, F);
  norms(3, 4096, 1, true, true, B, B, B);
  norms(3, 8000, 1, false, true, B, B, F);
  norms(3, 9000, 0, true, true, H, F, H);
  gate(20, 8, 2, 0, 1);
  gate(20, 200, 8, 1, 0);
  gate(5, 700, 40, 0, 0);
  std::printf("calls that returned an error: %d\n", failures);
  return failures ? 1 : 0;
}
