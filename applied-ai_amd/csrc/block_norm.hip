// The norms before and after a block of a transformer layer, fused with the block's gate and the residual sum, and their
// gradients. y is the block's output, res the residual stream in front of it:
//   n = y / sqrt(mean(y^2) + eps) * w_post      (or n = y)
//   h = alpha * res + beta * gate * n           the stream behind the block (gate: one value per channel, per row, or none)
//   z = h / sqrt(mean(h^2) + eps) * w_pre       what the next block reads
// With r = 1 / sqrt(mean(v^2) + eps), the gradient through v * r * w is r * (g w - v r^2 mean(g w v)).
//
// Bound by memory: a row is read once into registers, both norms' sums are taken over it there, and everything is written once (in the
// backward pass up to 4096 columns; what becomes of wider rows stands there). Sums are fp32; z is
// computed from the sum before it is rounded to the stream's type. The backward pass starts from the stored stream and
// computes both norms' r again from the rows, which it reads anyway: nothing but the stream is kept between the passes.
// Gradients of weights and of a gate per channel are sums over rows: a workgroup adds up its rows in registers, the workgroups'
// sums are added in a fixed order by a second kernel (no atomics: the same inputs give the same bits).
#include "common.h"
#include "kernels.h"

namespace {

// A row is taken in pieces of eight elements, which may lie anywhere: the hardware's 16-byte loads and stores need no alignment.
// n below is how many of a piece's elements exist: 8 and more all of them, fewer only in the last piece of a width that is no
// multiple of 8, which is read and written by element.
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));

DEVINL const char* at(const void* p, bool wide, int64_t i) { return (const char*)p + (wide ? 4 * i : 2 * i); }
DEVINL char* at(void* p, bool wide, int64_t i) { return (char*)p + (wide ? 4 * i : 2 * i); }

// A piece as it is in memory: a row waits in registers in half the space of its floats where it has 16 bits.
template <bool WIDE> struct Raw {
  u32x4_t w[WIDE ? 2 : 1];
  DEVINL void clear() {
#pragma unroll
    for (int i = 0; i < (WIDE ? 2 : 1); ++i) w[i] = u32x4_t{0u, 0u, 0u, 0u};
  }
  DEVINL void load(const void* p, int i, int n) {
    const char* s = at(p, WIDE, i);
    if (n >= 8) {
      w[0] = *(const u32x4_any_t*)s;
      if (WIDE) w[WIDE] = *(const u32x4_any_t*)(s + 16);
      return;
    }
    clear();
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) {
        if (WIDE) w[WIDE * (e >> 2)][e & 3] = ((const uint32_t*)s)[e];
        else w[0][e >> 1] |= (uint32_t)((const uint16_t*)s)[e] << (16 * (e & 1));
      }
  }
  template <bool F16> DEVINL float get(int e) const {
    const uint32_t wide = w[WIDE * (e >> 2)][e & 3];
    if (WIDE) return __builtin_bit_cast(float, wide);
    return f32_of_16<F16>((uint16_t)(w[0][(e >> 1) & 3] >> (16 * (e & 1))));
  }
};

template <bool F16, bool WIDE> DEVINL void load_v(const void* p, int i, int n, float (&v)[8]) {
  Raw<WIDE> r;
  r.load(p, i, n);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = r.template get<F16>(e);
}
template <bool F16, bool WIDE> DEVINL void store_v(void* p, int i, int n, const float (&v)[8]) {
  char* s = at(p, WIDE, i);
  if (n >= 8) {
    if (WIDE) {
      *(f32x4_any_t*)s = f32x4_t{v[0], v[1], v[2], v[3]};
      *(f32x4_any_t*)(s + 16) = f32x4_t{v[4], v[5], v[6], v[7]};
    } else {
      *(u32x4_any_t*)s = u32x4_t{pack_16x2<F16>(v[0], v[1]), pack_16x2<F16>(v[2], v[3]), pack_16x2<F16>(v[4], v[5]), pack_16x2<F16>(v[6], v[7])};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < n) {
      if (WIDE) ((float*)s)[e] = v[e];
      else ((uint16_t*)s)[e] = cvt_16<F16>(v[e]);
    }
}
// Weights and gate are in 32 bits or in the rows' type: decided once per launch.
template <bool F16> DEVINL void load_w(const void* p, bool wide, int i, int n, float (&v)[8]) {
  if (wide) load_v<F16, true>(p, i, n, v);
  else load_v<F16, false>(p, i, n, v);
}
template <bool F16> DEVINL float load_one(const void* p, bool wide, int64_t i) {
  return wide ? ((const float*)p)[i] : f32_of_16<F16>(((const uint16_t*)p)[i]);
}

// Sums of N values over the TPR threads of a row; every thread gets them. red: one entry per wave of the workgroup; two
// calls in a row use two of them.
template <int TPR, int N> DEVINL void row_sums(float (&v)[N], float (*red)[N]) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], d, 64);
  if (TPR > 64) {
    if (lane_id() == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave_id()][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) v[i] += red[w][i];
    }
  }
}

__host__ __device__ inline int sums_pitch(int d) { return (d + 3) & ~3; }

// TPR threads to a row, NV pieces to a thread. TPR = 64: a workgroup has four rows.
// 8192 x 4096, both norms, fp32 stream (402 MB): 74 us, 5.5 TB/s; with 256 threads and two pieces each 78 us. 8 rows: 4.6 us.
template <bool F16, bool WIDE, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_norm_forward(NormParams p) {
  constexpr int RPB = TPR == 64 ? 4 : 1;
  __shared__ float red[2][TPR / 64][1];
  const int64_t t = (int64_t)blockIdx.x * RPB + (RPB > 1 ? wave_id() : 0);
  if (t >= p.T) return;
  const int tid = RPB > 1 ? lane_id() : threadIdx.x;
  // a thread's pieces lie TPR * 8 elements apart from its first one
  const int c0 = tid * 8, left = p.d - c0;
  const char* y_at = at(p.y, false, t * p.ldy + c0);
  const char* r_at = at(p.res, WIDE, t * p.ldr + c0);
  const char* w_post = at(p.w_post, p.wide_w, c0);
  const char* gate = at(p.gate, p.wide_w, c0);
  const char* w_pre = at(p.w_pre, p.wide_w, c0);
  char* h_at = at(p.h, WIDE, t * p.d + c0);
  char* z_at = at(p.z, false, t * p.d + c0);
  float y[NV][8], h[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    constexpr int STEP = TPR * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[i][e] = h[i][e] = 0.f;
    if (i * STEP < left) {
      if (p.y) load_v<F16, false>(y_at, i * STEP, left - i * STEP, y[i]);
      load_v<F16, WIDE>(r_at, i * STEP, left - i * STEP, h[i]);
    }
  }
  if (p.y) {
    float ry = 1.f;
    if (p.w_post) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[0] += y[i][e] * y[i][e];
      row_sums<TPR>(s, red[0]);
      ry = 1.f / sqrtf(s[0] / (float)p.d + p.eps);
    }
    const float row_gate = p.beta * (p.gate && p.gate_kind == 2 ? load_one<F16>(p.gate, p.wide_w, t) : 1.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int STEP = TPR * 8;
      if (i * STEP < left) {
        float w[8], g[8];
        if (p.w_post) load_w<F16>(w_post, p.wide_w, i * STEP, left - i * STEP, w);
        if (p.gate && p.gate_kind == 1) load_w<F16>(gate, p.wide_w, i * STEP, left - i * STEP, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float n = y[i][e];
          if (p.w_post) n = n * ry * w[e];
          if (p.gate && p.gate_kind == 1) n *= g[e];
          h[i][e] = p.alpha * h[i][e] + row_gate * n;
        }
        store_v<F16, WIDE>(h_at, i * STEP, left - i * STEP, h[i]);
      }
    }
  }
  if (!p.w_pre) return;
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] += h[i][e] * h[i][e];
  row_sums<TPR>(s, red[1]);
  const float rh = 1.f / sqrtf(s[0] / (float)p.d + p.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    constexpr int STEP = TPR * 8;
    if (i * STEP < left) {
      float w[8];
      load_w<F16>(w_pre, p.wide_w, i * STEP, left - i * STEP, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = h[i][e] * rh * w[e];
      store_v<F16, false>(z_at, i * STEP, left - i * STEP, w);
    }
  }
}

// Rows blockIdx.x * RPB + ..., in steps of the grid; the next row is on its way while one is worked on.
// sums [3][parts][d rounded up to four]: the workgroups' (TPR = 64: waves') shares of the gradients of w_pre, w_post and a
// channel gate, each only where it is asked for.
// The hardware counts a wave's loads and stores in one order, so that waiting for one waits for all before it. For the next row's
// loads to stay in flight over a whole row, nothing else is loaded from memory in between: a thread keeps its columns' weights
// and gate in LDS (KEEP, where they fit in 64 KB); and the stores behind them are the same in number on every path (FULL: every
// thread has NV whole pieces of the row), so that the wait for the loads need not wait for them.
// HAS_Y false: the norm alone.
// 4096 x 4096 bf16 with a channel gate (201 MB and 25 MB of shares, of which the counters see 92 MB written, as they should): 42 us;
// without the LDS copies 63, with 512 threads to a row 51, without the row in advance 46.
// Wider rows are not as fast. Beyond 4096 columns the LDS copies are off (counted at 32 bits they take more than 64 KB) and weights
// come from memory for every row; two pieces of a row that is not 8192 wide spill 14 to 52 registers, and the 128 registers of
// each of 1024 threads do not hold two pieces: 134 to 277 go to scratch (without y 10, of an fp32 stream). 4096 rows of 5120
// columns 98 us, 7168 121, 8192 115, 12288 369, 16384 613: 2.9 to 3.9 and 1.8 to 1.5 TB/s with the shares.
template <bool F16, bool WIDE, int TPR, int NV, bool HAS_Y, bool FULL>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, TPR == 1024 ? 4 : 2) void block_norm_backward(NormGradParams p) {
  constexpr int RPB = TPR == 64 ? 4 : 1, STEP = TPR * 8, THREADS = TPR > 256 ? TPR : 256;
  constexpr bool AHEAD = TPR < 1024;  // the widest rows leave no registers for a second one, nor for all of the first
  constexpr bool KEEP = 3 * NV * THREADS * 32 <= 65536;
  __shared__ float red3[2][TPR / 64][3];
  __shared__ float red2[2][TPR / 64][2];
  extern __shared__ u32x4_t kept[];  // [3][NV][1 or 2][THREADS]: w_pre, w_post, gate
  const int tid = RPB > 1 ? lane_id() : threadIdx.x;
  const int part = blockIdx.x * RPB + (RPB > 1 ? wave_id() : 0);
  const int64_t next = (int64_t)gridDim.x * RPB;
  const float inv_d = 1.f / (float)p.d;
  const int c0 = tid * 8, left = p.d - c0;
  const bool post = HAS_Y && p.w_post, channel = HAS_Y && p.gate_kind == 1;
  auto there = [&](int i) { return FULL || i * STEP < left; };
  auto rest = [&](int i) { return FULL ? 8 : left - i * STEP; };
  const int planes = p.wide_w ? 2 : 1;
  auto keep = [&](int k, const void* w) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (there(i)) {
        u32x4_t* d = kept + (k * NV + i) * planes * THREADS + threadIdx.x;
        if (p.wide_w) {
          Raw<true> r;
          r.load(at(w, true, c0), i * STEP, rest(i));
          d[0] = r.w[0];
          d[THREADS] = r.w[1];
        } else {
          Raw<false> r;
          r.load(at(w, false, c0), i * STEP, rest(i));
          d[0] = r.w[0];
        }
      }
  };
  auto weight = [&](int k, const void* w, int i, float (&v)[8]) {
    if (!KEEP) return load_w<F16>(at(w, p.wide_w, c0), p.wide_w, i * STEP, rest(i), v);
    const u32x4_t* s = kept + (k * NV + i) * planes * THREADS + threadIdx.x;
    if (p.wide_w) {
      Raw<true> r;
      r.w[0] = s[0];
      r.w[1] = s[THREADS];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = r.template get<F16>(e);
    } else {
      Raw<false> r;
      r.w[0] = s[0];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = r.template get<F16>(e);
    }
  };
  if (KEEP) {
    if (p.w_pre) keep(0, p.w_pre);
    if (post) keep(1, p.w_post);
    if (channel) keep(2, p.gate);
  }
  float a_pre[NV][8], a_post[NV][8], a_gate[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) a_pre[i][e] = a_post[i][e] = a_gate[i][e] = 0.f;
  Raw<false> y[NV], gz[NV], y2[NV], gz2[NV];
  Raw<WIDE> h[NV], gh[NV], h2[NV], gh2[NV];
  auto load = [&](int64_t t) {
    const char* y_at = at(p.y, false, t * p.ldy + c0);
    const char* h_at = at(p.h, WIDE, t * p.ldh + c0);
    const char* gh_at = at(p.gh, WIDE, t * p.ldgh + c0);
    const char* gz_at = at(p.gz, false, t * p.ldgz + c0);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (there(i)) {
        if (HAS_Y) y2[i].load(y_at, i * STEP, rest(i));
        if (p.gh) gh2[i].load(gh_at, i * STEP, rest(i));
        if (p.w_pre) {
          h2[i].load(h_at, i * STEP, rest(i));
          gz2[i].load(gz_at, i * STEP, rest(i));
        }
      }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) y2[i].clear(), gz2[i].clear(), h2[i].clear(), gh2[i].clear();
  if (AHEAD && part < p.T) load(part);
  int turn = 0;
  for (int64_t t = part; t < p.T; t += next, turn ^= 1) {
    if (!AHEAD) load(t);
#pragma unroll
    for (int i = 0; i < NV; ++i) y[i] = y2[i], gz[i] = gz2[i], h[i] = h2[i], gh[i] = gh2[i];
    if (AHEAD && t + next < p.T) load(t + next);
    float s3[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (there(i)) {
        if (p.w_pre) {
          float w[8];
          weight(0, p.w_pre, i, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = h[i].template get<F16>(e);
            s3[0] += v * v;
            s3[1] += gz[i].template get<F16>(e) * w[e] * v;
          }
        }
        if (HAS_Y)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = y[i].template get<F16>(e);
            s3[2] += v * v;
          }
      }
    wave_whole();
    row_sums<TPR>(s3, red3[turn]);
    const float rh = 1.f / sqrtf(s3[0] * inv_d + p.eps), ry = post ? 1.f / sqrtf(s3[2] * inv_d + p.eps) : 1.f;
    const float dot_h = s3[1] * inv_d * rh * rh;
    const float row_gate = p.gate_kind == 2 ? load_one<F16>(p.gate, p.wide_w, t) : 1.f;
    char* gres = at(p.gres, WIDE, t * p.d + c0);
    float g[NV][8];  // the gradient of the stream, then that of the normed y
    float s2[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (there(i)) {
        float w[8], gt[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[i][e] = gh[i].template get<F16>(e);
        if (p.w_pre) {
          weight(0, p.w_pre, i, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = h[i].template get<F16>(e), z = gz[i].template get<F16>(e);
            g[i][e] += rh * (z * w[e] - v * dot_h);
            a_pre[i][e] += z * v * rh;
          }
        }
        float gr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) gr[e] = p.alpha * g[i][e];
        store_v<F16, WIDE>(gres, i * STEP, rest(i), gr);
        if (HAS_Y) {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = 1.f, gt[e] = row_gate;
          if (post) weight(1, p.w_post, i, w);
          if (channel) weight(2, p.gate, i, gt);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float b = p.beta * g[i][e];                       // gradient of gate * n
            const float v = y[i].template get<F16>(e), yn = v * ry;  // n = yn * w
            a_gate[i][e] += b * yn * w[e];
            a_post[i][e] += b * gt[e] * yn;
            s2[0] += b * yn * w[e];
            g[i][e] = b * gt[e] * w[e];                             // gradient of yn
            s2[1] += g[i][e] * v;
          }
        }
      }
    if (!HAS_Y) continue;
    wave_whole();
    if (post || p.gate_kind == 2) row_sums<TPR>(s2, red2[turn]);
    if (p.gate_kind == 2) {
      // the sum over a row is this row's gradient; the channel sums are not used
      if (tid == 0) {
        if (p.wide_w) ((float*)p.g_gate)[t] = s2[0];
        else ((uint16_t*)p.g_gate)[t] = cvt_16<F16>(s2[0]);
      }
    }
    const float dot_y = post ? s2[1] * inv_d * ry * ry : 0.f;
    char* gy = at(p.gy, false, t * p.d + c0);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (there(i)) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = ry * (g[i][e] - y[i].template get<F16>(e) * dot_y);
        store_v<F16, false>(gy, i * STEP, rest(i), o);
      }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (there(i)) {
      float* sums = p.sums + (int64_t)part * sums_pitch(p.d) + c0;
      const int64_t which = (int64_t)p.parts * sums_pitch(p.d);
      if (p.w_pre) store_v<F16, true>(sums, i * STEP, rest(i), a_pre[i]);
      if (post) store_v<F16, true>(sums + which, i * STEP, rest(i), a_post[i]);
      if (channel) store_v<F16, true>(sums + 2 * which, i * STEP, rest(i), a_gate[i]);
    }
}

// out[c] = sum over parts of sums[which][part][c]: 32 columns, four to a thread, and 32 strands of parts to a workgroup; the
// strands are added in order. (The pitch of sums is d rounded up to four; what lies between is read and not used.)
template <bool F16>
__global__ __launch_bounds__(256) void block_norm_sums(NormGradParams p) {
  __shared__ float red[32][32];
  const int which = blockIdx.y;
  void* out = which == 0 ? p.g_pre : which == 1 ? p.g_post : p.gate_kind == 1 ? p.g_gate : nullptr;
  if (!out) return;
  const int quad = threadIdx.x & 7, strand = threadIdx.x >> 3, c = blockIdx.x * 32 + 4 * quad;
  const int pitch = sums_pitch(p.d);
  const float* at = p.sums + (int64_t)which * p.parts * pitch + c;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int i = strand; i < p.parts; i += 32 * 8) {
    f32x4_t a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
      a[j] = c < p.d ? *(const f32x4_t*)(at + (int64_t)min(i + 32 * j, p.parts - 1) * pitch) : zero;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + 32 * j < p.parts) v += a[j];
  }
  *(f32x4_t*)&red[strand][4 * quad] = v;
  __syncthreads();
  const int col = blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x < 32 && col < p.d) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x];
    if (p.wide_w) ((float*)out)[col] = s;
    else ((uint16_t*)out)[col] = cvt_16<F16>(s);
  }
}

// Gates of rows without columns have gradients of zero.
__global__ __launch_bounds__(256) void block_norm_no_columns(void* g_gate, bool wide, int T) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  if (wide) ((float*)g_gate)[t] = 0.f;
  else ((uint16_t*)g_gate)[t] = 0;
}

// Threads to a row and pieces to a thread by width: a wave up to 512 columns (1024 in the forward pass), else as many threads
// as keep a row in registers.
template <bool F16, bool WIDE>
void forward(const NormParams& p, hipStream_t stream) {
#define LAUNCH(TPR, NV)                                                                                                      \
  hipLaunchKernelGGL((block_norm_forward<F16, WIDE, TPR, NV>), dim3((unsigned)((TPR) == 64 ? (p.T + 3) / 4 : p.T)),           \
                     dim3((TPR) > 256 ? (TPR) : 256), 0, stream, p)
  if (p.d <= 512) LAUNCH(64, 1);
  else if (p.d <= 1024) LAUNCH(64, 2);
  else if (p.d <= 2048) LAUNCH(256, 1);
  else if (p.d <= 4096) LAUNCH(512, 1);
  else if (p.d <= 8192) LAUNCH(512, 2);
  else LAUNCH(512, 4);
#undef LAUNCH
}

template <bool F16, bool WIDE, int TPR, int NV>
void launch_backward(const NormGradParams& p, int grid, hipStream_t stream) {
  constexpr int THREADS = TPR > 256 ? TPR : 256;
  const size_t lds = 3 * NV * THREADS * 32 <= 65536 ? (size_t)3 * NV * THREADS * (p.wide_w ? 32 : 16) : 0;
  if (!p.y) hipLaunchKernelGGL((block_norm_backward<F16, WIDE, TPR, NV, false, false>), dim3(grid), dim3(THREADS), lds, stream, p);
  else if (p.d == TPR * NV * 8) hipLaunchKernelGGL((block_norm_backward<F16, WIDE, TPR, NV, true, true>), dim3(grid), dim3(THREADS), lds, stream, p);
  else hipLaunchKernelGGL((block_norm_backward<F16, WIDE, TPR, NV, true, false>), dim3(grid), dim3(THREADS), lds, stream, p);
}

template <bool F16, bool WIDE>
void backward(const NormGradParams& p, int grid, hipStream_t stream) {
  if (p.d <= 512) launch_backward<F16, WIDE, 64, 1>(p, grid, stream);
  else if (p.d <= 2048) launch_backward<F16, WIDE, 256, 1>(p, grid, stream);
  else if (p.d <= 4096) launch_backward<F16, WIDE, 256, 2>(p, grid, stream);
  else if (p.d <= 8192) launch_backward<F16, WIDE, 512, 2>(p, grid, stream);
  else launch_backward<F16, WIDE, 1024, 2>(p, grid, stream);
}

// Workgroups of the backward pass: two to a CU, and what a workgroup's partial sums cost stays small beside its rows.
int rows_per_group(int d) { return d <= 512 ? 4 : 1; }
int grad_grid(int64_t T, int d) {
  const int64_t want = (T + rows_per_group(d) - 1) / rows_per_group(d);
  return (int)(want < 512 ? want : 512);
}
int grad_parts(int64_t T, int d) { return grad_grid(T, d) * rows_per_group(d); }

}  // namespace

size_t block_norm_backward_workspace(int64_t T, int d) { return (size_t)3 * grad_parts(T, d) * sums_pitch(d) * sizeof(float); }

hipError_t block_norm_launch(const NormParams& p, bool fp16, hipStream_t stream) {
  if (fp16) p.wide ? forward<true, true>(p, stream) : forward<true, false>(p, stream);
  else p.wide ? forward<false, true>(p, stream) : forward<false, false>(p, stream);
  return hipGetLastError();
}

hipError_t block_norm_backward_launch(NormGradParams p, bool fp16, hipStream_t stream) {
  if (p.d == 0) {
    if (p.T > 0 && p.gate_kind == 2) hipLaunchKernelGGL(block_norm_no_columns, dim3((p.T + 255) / 256), dim3(256), 0, stream, p.g_gate, p.wide_w, p.T);
    return hipGetLastError();
  }
  const int grid = grad_grid(p.T, p.d);
  p.parts = grad_parts(p.T, p.d);
  if (p.T > 0) {  // else the sums below are zeros
    if (fp16) p.wide ? backward<true, true>(p, grid, stream) : backward<true, false>(p, grid, stream);
    else p.wide ? backward<false, true>(p, grid, stream) : backward<false, false>(p, grid, stream);
  }
  if (p.g_pre || p.g_post || (p.gate_kind == 1 && p.g_gate)) {
    const dim3 g((unsigned)((p.d + 31) / 32), 3);
    if (fp16) hipLaunchKernelGGL((block_norm_sums<true>), g, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((block_norm_sums<false>), g, dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}
