// The router's gate: the k best experts of a row with the weights of their rows in the layer's sum, and its gradient.
//
//   softmax:  p_e = exp(l_e) / sum_i exp(l_i)         sigmoid:  p_e = 1 / (1 + exp(-l_e))
//   ids = the k largest logits, descending, ties to the lower expert (both scores grow with the logit)
//   weight_j = scale * p_{ids_j}, with renormalisation divided by sum_j p_{ids_j}
//
// Renormalised weights are the softmax of log p over the chosen experts, which needs neither the whole row's sum (softmax:
// log p = l up to a constant of the row) nor a p that has not underflowed (sigmoid: log p = min(l, 0) - log(1 + exp(-|l|))).
// A row whose chosen logits are all -infinity gets weights and gradients of zero.
// The gradient with g the gradient of the weights and w = weight / scale:
//   renormalised  d log p_j = scale * w_j (g_j - sum_i w_i g_i);  softmax: dl = d log p, sigmoid: dl = (1 - p) d log p
//   softmax       dl_e = scale * p_e (g_e - sum_j g_j w_j), g_e = 0 for experts not chosen
//   sigmoid       dl_j = scale * p_j (1 - p_j) g_j
//
// Bound by latency at these sizes (a row is at most 3 KB): rows are spread over few lanes, so that a wave has several of them in
// flight (launch_size below).
#include "common.h"
#include "kernels.h"

namespace {

DEVINL float load_logit(const void* logits, int dtype, int64_t i) {
  if (dtype == 2) return ((const float*)logits)[i];
  const uint16_t h = ((const uint16_t*)logits)[i];
  return dtype == 1 ? f32_of_16<true>(h) : f32_of_16<false>(h);
}
DEVINL void store_logit(void* out, int dtype, int64_t i, float v) {
  if (dtype == 2) ((float*)out)[i] = v;
  else ((uint16_t*)out)[i] = dtype == 1 ? cvt_16<true>(v) : cvt_16<false>(v);
}
DEVINL float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }
DEVINL float log_sigmoid(float l) { return min(l, 0.f) - log1pf(expf(-__builtin_fabsf(l))); }

template <int LANES> DEVINL float row_max(float v) {
#pragma unroll
  for (int d = LANES / 2; d >= 1; d >>= 1) v = max(v, __shfl_xor(v, d, 64));
  return v;
}
template <int LANES> DEVINL float row_sum(float v) {
#pragma unroll
  for (int d = LANES / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// The weights over scale of the chosen experts, one per lane j < k (l: its logit), and the row's softmax terms where they are
// needed. all: the row's logits, PER in a lane.
template <int LANES, int PER, bool SIGMOID, bool RENORM>
DEVINL float chosen_weight(float l, bool mine, const float (&all)[PER], float& row_m, float& row_s) {
  if (RENORM) {
    const float lp = !mine ? -__builtin_inff() : SIGMOID ? log_sigmoid(l) : l;
    const float m = row_max<LANES>(lp);
    const float e = mine && m > -__builtin_inff() ? expf(lp - m) : lp != lp ? lp : 0.f;
    const float s = row_sum<LANES>(e);
    return s == 0.f ? 0.f : e / s;
  }
  if (SIGMOID) return mine ? sigmoid(l) : 0.f;
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) m = max(m, all[i]);
  row_m = row_max<LANES>(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) s += row_m > -__builtin_inff() ? expf(all[i] - row_m) : all[i] != all[i] ? all[i] : 0.f;
  row_s = row_sum<LANES>(s);
  return mine && row_s != 0.f ? expf(l - row_m) / row_s : 0.f;
}

template <int LANES, int PER, bool SIGMOID, bool RENORM>
__global__ __launch_bounds__(256) void gate_forward(GateParams p) {
  constexpr int ROWS = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int t = blockIdx.x * ROWS + threadIdx.x / LANES;
  const bool live = t < p.T;
  const int64_t row = (int64_t)(live ? t : p.T - 1) * p.E;
  // A logit as an unsigned number of the same order: 0 for what is not there or taken, 1 for NaN. -0 counts as 0.
  float v[PER];
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + LANES * i;
    v[i] = e < p.E ? load_logit(p.logits, p.dtype, row + e) : -__builtin_inff();
    const uint32_t u = __builtin_bit_cast(uint32_t, v[i] + 0.f);
    key[i] = e >= p.E ? 0u : v[i] != v[i] ? 1u : u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
  }
  const int first_lane = (threadIdx.x & 63) & ~(LANES - 1);
  constexpr unsigned long long ROW = LANES == 64 ? ~0ull : (1ull << (LANES & 63)) - 1;
  float my_l = -__builtin_inff();
  for (int j = 0; j < p.k; ++j) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) best = max(best, key[i]);
#pragma unroll
    for (int d = LANES / 2; d >= 1; d >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, d, 64));
    // who holds it; of equal ones the lowest expert
    uint32_t at = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) at |= (key[i] == best ? 1u : 0u) << i;
    int e = at ? lane + LANES * __builtin_ctz(at) : 0x7fffffff;
    const unsigned long long holders = (__ballot(at != 0) >> first_lane) & ROW;
    bool mine = at != 0;
    if (__ballot(__popcll(holders) > 1)) {
      int low = e;
#pragma unroll
      for (int d = LANES / 2; d >= 1; d >>= 1) low = min(low, __shfl_xor(low, d, 64));
      mine = e == low;
    }
    wave_whole();
    if (mine) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (e == lane + LANES * i) key[i] = 0;
      if (live) p.ids[(int64_t)t * p.k + j] = e;
    }
    wave_whole();
    const uint32_t u = best >> 31 ? best ^ 0x80000000u : ~best;
    if (lane == j) my_l = best == 1u ? __builtin_nanf("") : __builtin_bit_cast(float, u);
  }
  float m, s;
  const float w = chosen_weight<LANES, PER, SIGMOID, RENORM>(my_l, lane < p.k, v, m, s);
  if (live && lane < p.k) p.weights[(int64_t)t * p.k + lane] = p.scale * w;
}

// ids outside [0, E) have no logit: they take no part.
template <int LANES, int PER, bool SIGMOID, bool RENORM>
__global__ __launch_bounds__(256) void gate_backward(GateParams p) {
  constexpr int ROWS = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  const int t = blockIdx.x * ROWS + threadIdx.x / LANES;
  const bool live = t < p.T;
  const int64_t row = (int64_t)(live ? t : p.T - 1) * p.E;
  const int64_t at = (int64_t)(live ? t : p.T - 1) * p.k + lane;
  const int id = lane < p.k ? p.ids[at] : -1;
  const bool mine = id >= 0 && id < p.E;
  const float l = mine ? load_logit(p.logits, p.dtype, row + id) : -__builtin_inff();
  const float g = mine ? p.weights[at] : 0.f;
  float v[PER];
  if (!SIGMOID && !RENORM) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + LANES * i;
      v[i] = e < p.E ? load_logit(p.logits, p.dtype, row + e) : -__builtin_inff();
    }
  }
  float m = 0.f, s = 0.f;
  const float w = chosen_weight<LANES, PER, SIGMOID, RENORM>(l, mine, v, m, s);
  const float dot = row_sum<LANES>(mine ? w * g : 0.f);
  float d = RENORM ? p.scale * w * (g - dot) : p.scale * w * g;
  if (SIGMOID) d *= sigmoid(-l);
  if (!mine || l == -__builtin_inff()) d = 0.f;  // also where sigmoid(-l) is 0 * infinity
  float o[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = !SIGMOID && !RENORM && s != 0.f && v[i] > -__builtin_inff() ? -p.scale * dot * (expf(v[i] - m) / s) : 0.f;
  for (int j = 0; j < p.k; ++j) {
    const float dj = __shfl(d, (threadIdx.x & 63 & ~(LANES - 1)) + j, 64);
    const int ej = __shfl(mine ? id : -1, (threadIdx.x & 63 & ~(LANES - 1)) + j, 64);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (ej == lane + LANES * i) o[i] += dj;
  }
  if (live)
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + LANES * i < p.E) store_logit(p.grad_logits, p.dtype, row + lane + LANES * i, o[i]);
}

template <int LANES, int PER, bool SIGMOID, bool RENORM>
void launch(const GateParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.T + 256 / LANES - 1) / (256 / LANES))), block(256);
  if (p.grad_logits) hipLaunchKernelGGL((gate_backward<LANES, PER, SIGMOID, RENORM>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((gate_forward<LANES, PER, SIGMOID, RENORM>), grid, block, 0, stream, p);
}

// Lanes to a row: a selection is a search in a lane's experts and a reduction over the row's lanes; a few lanes need fewer rounds
// of it, and do several rows at once. Lane j holds the j-th choice's weight, so there are at least k of them. Rows of 256
// experts, 8 chosen of sigmoid, with 16, 32 and 64 lanes in a captured graph: 64 rows 8.4, 7.0 and 6.6 us, 4096 rows 8.6, 7.5 and 7.3,
// 32768 rows 21.8, 25.0 and 32.2: 32 are within 10 % of the best for few rows and 15 % for many.
template <bool SIGMOID, bool RENORM>
void launch_size(const GateParams& p, hipStream_t stream) {
  if (p.k <= 8 && p.E <= 8) launch<8, 1, SIGMOID, RENORM>(p, stream);
  else if (p.k <= 16 && p.E <= 16) launch<16, 1, SIGMOID, RENORM>(p, stream);
  else if (p.k <= 16 && p.E <= 64) launch<16, 4, SIGMOID, RENORM>(p, stream);
  else if (p.k <= 32 && p.E <= 256) launch<32, 8, SIGMOID, RENORM>(p, stream);
  else if (p.E <= 64) launch<64, 1, SIGMOID, RENORM>(p, stream);
  else if (p.E <= 256) launch<64, 4, SIGMOID, RENORM>(p, stream);
  else launch<64, 12, SIGMOID, RENORM>(p, stream);
}

}  // namespace

hipError_t gate_launch(const GateParams& p, bool sigmoid, bool renormalize, hipStream_t stream) {
  if (sigmoid) renormalize ? launch_size<true, true>(p, stream) : launch_size<true, false>(p, stream);
  else renormalize ? launch_size<false, true>(p, stream) : launch_size<false, false>(p, stream);
  return hipGetLastError();
}
