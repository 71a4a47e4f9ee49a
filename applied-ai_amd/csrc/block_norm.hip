// The norms before and after a block of a transformer layer, fused with the block's gate and the residual sum, and their
// gradients. y is the block's output, res the residual stream in front of it:
//   n = y / sqrt(mean(y^2) + eps) * w_post      (or n = y)
//   h = alpha * res + beta * gate * n           the stream behind the block (gate: one value per channel, per row, or none)
//   z = h / sqrt(mean(h^2) + eps) * w_pre       what the next block reads
// With r = 1 / sqrt(mean(v^2) + eps), the gradient through v * r * w is r * (g w - v r^2 mean(g w v)).
//
// Bound by memory: a row is read once into registers (8 elements of 16 bits to a load, V = 1 where the width or a pointer
// does not allow that), both norms' sums are taken over it there, and everything is written once. Sums are fp32; z is
// computed from the sum before it is rounded to the stream's type. The backward pass starts from the stored stream and
// computes both norms' r again from the rows, which it reads anyway: nothing but the stream is kept between the passes.
// Gradients of weights and of a gate per channel are sums over rows: a workgroup adds up its rows in registers, the workgroups'
// sums are added in a fixed order by a second kernel (no atomics: the same inputs give the same bits).
#include "common.h"
#include "kernels.h"

namespace {

// V elements at p as floats; WIDE: fp32, else 16 bits.
DEVINL const char* at(const void* p, bool wide, int64_t i) { return (const char*)p + (wide ? 4 * i : 2 * i); }
DEVINL char* at(void* p, bool wide, int64_t i) { return (char*)p + (wide ? 4 * i : 2 * i); }
template <int V, bool F16, bool WIDE> DEVINL void load_v(const void* p, int i, float (&v)[V]) {
  if (WIDE) {
    const float* s = (const float*)p + i;
    if (V == 1) {
      v[0] = s[0];
    } else {
#pragma unroll
      for (int b = 0; b < V / 4; ++b) {
        const f32x4_t q = ((const f32x4_t*)s)[b];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * b + e] = q[e];
      }
    }
  } else {
    const uint16_t* s = (const uint16_t*)p + i;
    if (V == 1) {
      v[0] = f32_of_16<F16>(s[0]);
    } else {
      const u32x4_t q = *(const u32x4_t*)s;
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = f32_of_16<F16>((uint16_t)(q[e >> 1] >> (16 * (e & 1))));
    }
  }
}
template <int V, bool F16, bool WIDE> DEVINL void store_v(void* p, int i, const float (&v)[V]) {
  if (WIDE) {
    float* s = (float*)p + i;
    if (V == 1) {
      s[0] = v[0];
    } else {
#pragma unroll
      for (int b = 0; b < V / 4; ++b) ((f32x4_t*)s)[b] = f32x4_t{v[4 * b], v[4 * b + 1], v[4 * b + 2], v[4 * b + 3]};
    }
  } else {
    uint16_t* s = (uint16_t*)p + i;
    if (V == 1) {
      s[0] = cvt_16<F16>(v[0]);
    } else {
      u32x4_t q;
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = pack_16x2<F16>(v[2 * e], v[2 * e + 1]);
      *(u32x4_t*)s = q;
    }
  }
}
// Weights and gate are in 32 bits or in the rows' type: decided once per launch.
template <int V, bool F16> DEVINL void load_w(const void* p, bool wide, int i, float (&v)[V]) {
  if (wide) load_v<V, F16, true>(p, i, v);
  else load_v<V, F16, false>(p, i, v);
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

// TPR threads to a row, NV pieces of V elements to a thread. TPR = 64: a workgroup has four rows.
template <bool F16, bool WIDE, int V, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_norm_forward(NormParams p) {
  constexpr int RPB = TPR == 64 ? 4 : 1;
  __shared__ float red[2][TPR / 64][1];
  const int64_t t = (int64_t)blockIdx.x * RPB + (RPB > 1 ? wave_id() : 0);
  if (t >= p.T) return;
  const int tid = RPB > 1 ? lane_id() : threadIdx.x;
  // a thread's pieces lie TPR * V elements apart from its first one
  const int c0 = tid * V, left = p.d - c0;
  const char* y_at = at(p.y, false, t * p.ldy + c0);
  const char* r_at = at(p.res, WIDE, t * p.ldr + c0);
  const char* w_post = at(p.w_post, p.wide_w, c0);
  const char* gate = at(p.gate, p.wide_w, c0);
  const char* w_pre = at(p.w_pre, p.wide_w, c0);
  char* h_at = at(p.h, WIDE, t * p.d + c0);
  char* z_at = at(p.z, false, t * p.d + c0);
  float y[NV][V], h[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    constexpr int STEP = TPR * V;
#pragma unroll
    for (int e = 0; e < V; ++e) y[i][e] = h[i][e] = 0.f;
    if (i * STEP < left) {
      if (p.y) load_v<V, F16, false>(y_at, i * STEP, y[i]);
      load_v<V, F16, WIDE>(r_at, i * STEP, h[i]);
    }
  }
  if (p.y) {
    float ry = 1.f;
    if (p.w_post) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += y[i][e] * y[i][e];
      row_sums<TPR>(s, red[0]);
      ry = 1.f / sqrtf(s[0] / (float)p.d + p.eps);
    }
    const float row_gate = p.beta * (p.gate && p.gate_kind == 2 ? load_one<F16>(p.gate, p.wide_w, t) : 1.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int STEP = TPR * V;
      if (i * STEP < left) {
        float w[V], g[V];
        if (p.w_post) load_w<V, F16>(w_post, p.wide_w, i * STEP, w);
        if (p.gate && p.gate_kind == 1) load_w<V, F16>(gate, p.wide_w, i * STEP, g);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float n = y[i][e];
          if (p.w_post) n = n * ry * w[e];
          if (p.gate && p.gate_kind == 1) n *= g[e];
          h[i][e] = p.alpha * h[i][e] + row_gate * n;
        }
        store_v<V, F16, WIDE>(h_at, i * STEP, h[i]);
      }
    }
  }
  if (!p.w_pre) return;
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) s[0] += h[i][e] * h[i][e];
  row_sums<TPR>(s, red[1]);
  const float rh = 1.f / sqrtf(s[0] / (float)p.d + p.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    constexpr int STEP = TPR * V;
    if (i * STEP < left) {
      float w[V];
      load_w<V, F16>(w_pre, p.wide_w, i * STEP, w);
#pragma unroll
      for (int e = 0; e < V; ++e) w[e] = h[i][e] * rh * w[e];
      store_v<V, F16, false>(z_at, i * STEP, w);
    }
  }
}

// Rows blockIdx.x * RPB + ..., in steps of the grid. sums [3][parts][d]: the workgroups' (TPR = 64: waves') shares of the
// gradients of w_pre, w_post and a channel gate, each only where it is asked for.
template <bool F16, bool WIDE, int V, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_norm_backward(NormGradParams p) {
  constexpr int RPB = TPR == 64 ? 4 : 1;
  __shared__ float red3[2][TPR / 64][3];
  __shared__ float red2[2][TPR / 64][2];
  const int tid = RPB > 1 ? lane_id() : threadIdx.x;
  const int part = blockIdx.x * RPB + (RPB > 1 ? wave_id() : 0);
  const float inv_d = 1.f / (float)p.d;
  const int c0 = tid * V, left = p.d - c0;
  const char* w_post = at(p.w_post, p.wide_w, c0);
  const char* gate = at(p.gate, p.wide_w, c0);
  const char* w_pre = at(p.w_pre, p.wide_w, c0);
  float a_pre[NV][V], a_post[NV][V], a_gate[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) a_pre[i][e] = a_post[i][e] = a_gate[i][e] = 0.f;
  int turn = 0;
  for (int64_t t = part; t < p.T; t += (int64_t)gridDim.x * RPB, turn ^= 1) {
    const char* y_at = at(p.y, false, t * p.ldy + c0);
    const char* h_at = at(p.h, WIDE, t * p.ldh + c0);
    const char* gh_at = at(p.gh, WIDE, t * p.ldgh + c0);
    const char* gz_at = at(p.gz, false, t * p.ldgz + c0);
    char* gres = at(p.gres, WIDE, t * p.d + c0);
    char* gy = at(p.gy, false, t * p.d + c0);
    float y[NV][V], h[NV][V], gh[NV][V], gz[NV][V];
    float s3[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int STEP = TPR * V;
#pragma unroll
      for (int e = 0; e < V; ++e) y[i][e] = h[i][e] = gh[i][e] = gz[i][e] = 0.f;
      if (i * STEP < left) {
        if (p.y) load_v<V, F16, false>(y_at, i * STEP, y[i]);
        if (p.gh) load_v<V, F16, WIDE>(gh_at, i * STEP, gh[i]);
        if (p.w_pre) {
          load_v<V, F16, WIDE>(h_at, i * STEP, h[i]);
          load_v<V, F16, false>(gz_at, i * STEP, gz[i]);
          float w[V];
          load_w<V, F16>(w_pre, p.wide_w, i * STEP, w);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            s3[0] += h[i][e] * h[i][e];
            s3[1] += gz[i][e] * w[e] * h[i][e];
          }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) s3[2] += y[i][e] * y[i][e];
      }
    }
    row_sums<TPR>(s3, red3[turn]);
    const float rh = 1.f / sqrtf(s3[0] * inv_d + p.eps), ry = p.w_post ? 1.f / sqrtf(s3[2] * inv_d + p.eps) : 1.f;
    const float dot_h = s3[1] * inv_d * rh * rh;
    const float row_gate = p.gate_kind == 2 ? load_one<F16>(p.gate, p.wide_w, t) : 1.f;
    float s2[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int STEP = TPR * V;
      if (i * STEP < left) {
        float w[V], g[V];
        if (p.w_pre) {
          load_w<V, F16>(w_pre, p.wide_w, i * STEP, w);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            gh[i][e] += rh * (gz[i][e] * w[e] - h[i][e] * dot_h);
            a_pre[i][e] += gz[i][e] * h[i][e] * rh;
          }
        }
        float gr[V];
#pragma unroll
        for (int e = 0; e < V; ++e) gr[e] = p.alpha * gh[i][e];
        if (p.gres) store_v<V, F16, WIDE>(gres, i * STEP, gr);
        if (p.y) {
          if (p.w_post) load_w<V, F16>(w_post, p.wide_w, i * STEP, w);
          if (p.gate_kind == 1) load_w<V, F16>(gate, p.wide_w, i * STEP, g);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float b = p.beta * gh[i][e];          // gradient of gate * n
            const float yn = y[i][e] * ry;              // n = yn * w
            const float wn = p.w_post ? w[e] : 1.f, gn = p.gate_kind == 1 ? g[e] : row_gate;
            a_gate[i][e] += b * yn * wn;
            a_post[i][e] += b * gn * yn;
            s2[0] += b * yn * wn;
            gh[i][e] = b * gn * wn;                     // gradient of yn
            s2[1] += gh[i][e] * y[i][e];
          }
        }
      }
    }
    if (!p.y) continue;
    if (p.w_post || p.gate_kind == 2) row_sums<TPR>(s2, red2[turn]);
    if (p.gate_kind == 2) {
      // the sum over a row is this row's gradient; the channel sums are not used
      if (tid == 0) {
        if (p.wide_w) ((float*)p.g_gate)[t] = s2[0];
        else ((uint16_t*)p.g_gate)[t] = cvt_16<F16>(s2[0]);
      }
    }
    const float dot_y = p.w_post ? s2[1] * inv_d * ry * ry : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int STEP = TPR * V;
      if (i * STEP < left) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = ry * (gh[i][e] - y[i][e] * dot_y);
        store_v<V, F16, false>(gy, i * STEP, o);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    constexpr int STEP = TPR * V;
    if (i * STEP < left) {
      float* sums = p.sums + (int64_t)part * p.d + c0;
      const int64_t which = (int64_t)p.parts * p.d;
      if (p.w_pre) store_v<V, F16, true>(sums, i * STEP, a_pre[i]);
      if (p.w_post) store_v<V, F16, true>(sums + which, i * STEP, a_post[i]);
      if (p.gate_kind == 1) store_v<V, F16, true>(sums + 2 * which, i * STEP, a_gate[i]);
    }
  }
}

// out[c] = sum over parts of sums[which][part][c]: 64 columns and 16 strands of parts to a workgroup, the strands added in order.
template <bool F16>
__global__ __launch_bounds__(1024) void block_norm_sums(NormGradParams p) {
  __shared__ float red[16][64];
  const int which = blockIdx.y;
  void* out = which == 0 ? p.g_pre : which == 1 ? p.g_post : p.gate_kind == 1 ? p.g_gate : nullptr;
  if (!out) return;
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), strand = threadIdx.x >> 6;
  float s = 0.f;
  if (c < p.d)
    for (int i = strand; i < p.parts; i += 16) s += p.sums[((int64_t)which * p.parts + i) * p.d + c];
  red[strand][threadIdx.x & 63] = s;
  __syncthreads();
  if (strand == 0 && c < p.d) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i][threadIdx.x];
    if (p.wide_w) ((float*)out)[c] = s;
    else ((uint16_t*)out)[c] = cvt_16<F16>(s);
  }
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// Threads to a row and pieces to a thread by width: a wave up to 512 columns (1024 in the forward pass), else as many threads
// as keep a row's arrays in registers.
template <bool F16, bool WIDE, int V>
void forward(const NormParams& p, hipStream_t stream) {
  const int64_t n = (p.d + V - 1) / V;
#define LAUNCH(TPR, NV)                                                                                                      \
  hipLaunchKernelGGL((block_norm_forward<F16, WIDE, V, TPR, NV>), dim3((unsigned)((TPR) == 64 ? (p.T + 3) / 4 : p.T)),        \
                     dim3((TPR) > 256 ? (TPR) : 256), 0, stream, p)
  if constexpr (V == 8) {
    if (n <= 64) LAUNCH(64, 1);
    else if (n <= 128) LAUNCH(64, 2);
    else if (n <= 256) LAUNCH(256, 1);
    else if (n <= 512) LAUNCH(256, 2);
    else if (n <= 1024) LAUNCH(256, 4);
    else LAUNCH(512, 4);
  } else {
    if (n <= 256) LAUNCH(64, 4);
    else if (n <= 1024) LAUNCH(256, 4);
    else if (n <= 4096) LAUNCH(1024, 4);
    else if (n <= 8192) LAUNCH(1024, 8);
    else LAUNCH(1024, 16);
  }
#undef LAUNCH
}

template <bool F16, bool WIDE, int V>
void backward(const NormGradParams& p, int grid, hipStream_t stream) {
  const int64_t n = (p.d + V - 1) / V;
#define LAUNCH(TPR, NV)                                                                                                      \
  hipLaunchKernelGGL((block_norm_backward<F16, WIDE, V, TPR, NV>), dim3(grid), dim3((TPR) > 256 ? (TPR) : 256), 0, stream, p)
  if constexpr (V == 8) {
    if (n <= 64) LAUNCH(64, 1);
    else if (n <= 256) LAUNCH(256, 1);
    else if (n <= 512) LAUNCH(256, 2);
    else if (n <= 1024) LAUNCH(512, 2);
    else LAUNCH(1024, 2);
  } else {
    if (n <= 256) LAUNCH(64, 4);
    else if (n <= 1024) LAUNCH(256, 4);
    else if (n <= 4096) LAUNCH(1024, 4);
    else if (n <= 8192) LAUNCH(1024, 8);
    else LAUNCH(1024, 16);
  }
#undef LAUNCH
}

}  // namespace

// Workgroups of the backward pass: two to a CU, and what a workgroup's partial sums cost stays small beside its rows.
static int grad_grid(int64_t T, int d, bool vec) {
  const int rows = (vec ? d <= 512 : d <= 256) ? 4 : 1;
  const int64_t want = (T + rows - 1) / rows;
  return (int)(want < 512 ? want : 512);
}
static int grad_parts(int64_t T, int d, bool vec) { return grad_grid(T, d, vec) * ((vec ? d <= 512 : d <= 256) ? 4 : 1); }

size_t block_norm_backward_workspace(int64_t T, int d) {
  const int a = grad_parts(T, d, true), b = grad_parts(T, d, false);
  return (size_t)3 * (a > b ? a : b) * d * sizeof(float);
}

hipError_t block_norm_launch(const NormParams& p, bool fp16, hipStream_t stream) {
  const bool vec = p.d % 8 == 0 && p.ldy % 8 == 0 && p.ldr % 8 == 0 && aligned16(p.y) && aligned16(p.res) && aligned16(p.h) && aligned16(p.z) &&
                   aligned16(p.w_post) && aligned16(p.w_pre) && (p.gate_kind != 1 || aligned16(p.gate));
#define RUN(F16, WIDE) vec ? forward<F16, WIDE, 8>(p, stream) : forward<F16, WIDE, 1>(p, stream)
  if (fp16) p.wide ? (RUN(true, true)) : (RUN(true, false));
  else p.wide ? (RUN(false, true)) : (RUN(false, false));
#undef RUN
  return hipGetLastError();
}

hipError_t block_norm_backward_launch(NormGradParams p, bool fp16, hipStream_t stream) {
  const bool vec = p.d % 8 == 0 && p.ldy % 8 == 0 && p.ldh % 8 == 0 && p.ldgh % 8 == 0 && p.ldgz % 8 == 0 && aligned16(p.y) && aligned16(p.h) &&
                   aligned16(p.gh) && aligned16(p.gz) && aligned16(p.gy) && aligned16(p.gres) && aligned16(p.w_post) && aligned16(p.w_pre) &&
                   (p.gate_kind != 1 || aligned16(p.gate));
  const int grid = grad_grid(p.T, p.d, vec);
  p.parts = grad_parts(p.T, p.d, vec);
#define RUN(F16, WIDE) vec ? backward<F16, WIDE, 8>(p, grid, stream) : backward<F16, WIDE, 1>(p, grid, stream)
  if (p.T == 0) ;  // the sums below are then zeros
  else if (fp16) p.wide ? (RUN(true, true)) : (RUN(true, false));
  else p.wide ? (RUN(false, true)) : (RUN(false, false));
#undef RUN
  if (p.g_pre || p.g_post || (p.gate_kind == 1 && p.g_gate)) {
    const dim3 g((unsigned)((p.d + 63) / 64), 3);
    if (fp16) hipLaunchKernelGGL((block_norm_sums<true>), g, dim3(1024), 0, stream, p);
    else hipLaunchKernelGGL((block_norm_sums<false>), g, dim3(1024), 0, stream, p);
  }
  return hipGetLastError();
}
