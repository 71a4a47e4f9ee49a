// Low-rank adapters of many requests beside one shared projection, and their gradients.
//
// Row t of a batch names an adapter e = id(t) with matrices A_e [R, K] and B_e [N, R] and a factor s_e:
//   h[t] = A_e x[t]                     out[t] = y[t] + s_e B_e h[t]                 (rows without an adapter: out = y)
//   u[t] = s_e B_e^T gout[t]            gx[t] = gx_in[t] + A_e^T u[t]
//   gA_e = sum_t u[t] x[t]^T            gB_e = s_e sum_t gout[t] h[t]^T
// The rank R is small, so every product moves far more bytes than it computes: x, y, out, gout, gx pass once per kernel and
// the matrix instructions only keep up with memory. Three kernels do all of it:
//   shrink  [rows, C] . [R, C]^T  -> [rows, R]   the long axis C is reduced: split over workgroups and waves
//   expand  [rows, R] . [C, R]^T  -> [rows, C]   added to a row of y on its way through
//   wgrad   [rows, C]^T . [rows, R] -> [C, R]    rows are reduced, adapter by adapter
// and the backward pass runs shrink and expand on transposed copies of B and A (R x C each, small beside the rows).
//
// Rows are taken in adapter order (perm, offsets of the plan). Group g = adapter g for g < L and "no adapter" for g = L.
// A grid cannot know the groups' sizes without a copy to the host, so it counts slots of `unit` rows:
// group g owns slots [off_g / unit + g, off_{g+1} / unit + g + 1), at least as many as it needs, and a workgroup
// finds its group with one ballot over the group table (two beyond 64 groups). [rows, R] intermediates live in the same space
// with unit 16: group g's rows start at 16 * (off_g / 16 + g), so that every group is aligned and padded with zero rows.
//
// The intermediates are fp32. As matrix operands they are split into a high and a low part of the 16-bit type, which keep
// 16 (bf16) or 22 (fp16) significant bits: one matrix instruction covers 16 ranks, its 32-deep reduction holding
// [high 16 | low 16] against the same 16 columns of the other operand twice. For fp16 the rows are scaled by a power of two
// first, so that neither part leaves the type's range.
#include "common.h"
#include "kernels.h"

namespace {

typedef __attribute__((__vector_size__(2 * sizeof(uint16_t)))) uint16_t u16x2_t;
typedef short i16x4_t __attribute__((ext_vector_type(4)));

struct Rows {
  const int32_t* perm;     // [T] rows in group order
  const int32_t* offsets;  // [G + 1]
  int G;                   // adapters + 1
  int T;
};

DEVINL int clamp_off(const Rows& r, int g) { return min(max(r.offsets[g], 0), r.T); }

struct Slot {
  int group;   // -1: nothing here
  int first;   // position of the first row in perm
  int rows;    // 1 .. unit
  int padded;  // the same row's place among the 16-padded intermediates
  int begin;   // position of the group's first row
  int size;    // rows of the group
};

// Which rows slot v of `unit` rows holds. All lanes of the wave take part; the result is the same in all of them. Whatever
// the table holds, the rows named lie inside [0, T).
DEVINL Slot find_slot(const Rows& r, int v, int unit) {
  const int lane = lane_id();
  const int step = (r.G + 63) >> 6;
  int i = lane * step;
  bool le = i < r.G && clamp_off(r, min(i, r.G)) / unit + i <= v;
  int g = max(__popcll(__ballot(le)) - 1, 0) * step;
  if (step > 1) {
    i = g + lane;
    le = lane < step && i < r.G && clamp_off(r, min(i, r.G)) / unit + i <= v;
    g += max(__popcll(__ballot(le)) - 1, 0);
  }
  g = min(g, r.G - 1);
  Slot s;
  s.begin = clamp_off(r, g);
  s.size = clamp_off(r, g + 1) - s.begin;
  const int skip = (v - (s.begin / unit + g)) * unit;
  s.first = s.begin + skip;
  s.rows = min(unit, s.size - skip);
  s.padded = 16 * (s.begin / 16 + g) + skip;
  s.group = s.rows > 0 && skip >= 0 ? g : -1;
  return s;
}

DEVINL u32x4_t load16(const uint16_t* p) { return *(const u32x4_t*)p; }
// Eight elements p[0..7] of which only the first n exist; no alignment.
DEVINL u32x4_t load_some(const uint16_t* p, int n) {
  u32x4_t v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
  return v;
}

DEVINL float finite_max(float m, float v) {
  const float a = __builtin_fabsf(v);
  return a <= 3.4028234e38f ? max(m, a) : m;  // neither infinities nor NaN set a row's scale
}
// The power of two that brings a largest magnitude m to [2^13, 2^14), and its inverse: high in fp16's range, so that values
// far below the largest keep their bits.
DEVINL uint32_t scale_exponent(float m) { return min(max(__builtin_bit_cast(uint32_t, m) >> 23, 14u), 253u); }
DEVINL float pow2_down(float m) { return __builtin_bit_cast(float, (267u - scale_exponent(m)) << 23); }
DEVINL float pow2_up(float m) { return __builtin_bit_cast(float, (scale_exponent(m) - 13u) << 23); }
// v as high + low part of the 16-bit type; the low part of an infinity or NaN is 0.
template <bool F16> DEVINL void split16(float v, uint16_t& hi, uint16_t& lo) {
  hi = cvt_16<F16>(v);
  const float r = v - f32_of_16<F16>(hi);
  lo = __builtin_fabsf(r) <= 3.4028234e38f ? cvt_16<F16>(r) : (uint16_t)0;
}

// ---- shrink -------------------------------------------------------------------------------------------------------------
// part[split][padded row][r] = sum over the split's columns of x[row, c] * w[group, r, c].
// A workgroup takes MF x 16 rows and one split; its eight waves take an eighth of the split each and are summed through LDS.
// A lane holds 16 consecutive columns of its row as two operands: with the column order changed the same way on both sides
// the sum is the same, and four lanes read 128 consecutive bytes of a row.
struct ShrinkParams {
  const uint16_t* x;
  int64_t ldx;
  const uint16_t* w;  // [L, R, ldw]
  int64_t ldw;
  float* part;        // [S][P][Rp]
  Rows rows;
  int C, R, Rp, P, splits, per_wave;  // per_wave: columns per wave, a multiple of 64
};

template <bool F16, int NF, int MF, bool VEC>
__global__ __launch_bounds__(512) void lora_shrink(ShrinkParams p, int slots) {
  __shared__ f32x4_t red[4][MF * NF][64];
  const int split = blockIdx.x / slots;
  const Slot s = find_slot(p.rows, blockIdx.x - split * slots, 16 * MF);
  if (s.group < 0 || s.group == p.rows.G - 1) return;
  const int lane = lane_id(), wave = wave_id(), i16 = lane & 15, q = lane >> 4;
  const int mf = (s.rows + 15) >> 4;
  // Operand rows that do not exist read row 0 of their matrix: a result belongs to one row of each operand, and theirs are
  // not kept.
  const uint16_t* xr[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int t = p.rows.perm[s.first + min(16 * i + i16, s.rows - 1)];
    xr[i] = p.x + (int64_t)(t >= 0 && t < p.rows.T ? t : 0) * p.ldx + 16 * q;
  }
  const uint16_t* wr[NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int r = 16 * j + i16;
    wr[j] = p.w + ((int64_t)s.group * p.R + (r < p.R ? r : 0)) * p.ldw + 16 * q;
  }
  f32x4_t acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  auto multiply = [&](const u32x4_t (&xv)[MF][2], const u32x4_t (&wv)[NF][2]) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = mfma_16x16x32<F16>(xv[i][b], wv[j][b], acc[i][j]);
  };
  const int64_t begin = (int64_t)(split * 8 + wave) * p.per_wave;
  const int k1 = (int)min((int64_t)p.C, begin + p.per_wave);
  int k0 = (int)min(begin, (int64_t)p.C);
  if (VEC)
    for (; k0 + 64 <= k1; k0 += 64) {
      u32x4_t xv[MF][2], wv[NF][2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int j = 0; j < NF; ++j) wv[j][b] = load16(wr[j] + k0 + 8 * b);
#pragma unroll
        for (int i = 0; i < MF; ++i) xv[i][b] = load16(xr[i] + k0 + 8 * b);
      }
      multiply(xv, wv);
    }
  for (; k0 < k1; k0 += 64) {
    u32x4_t xv[MF][2], wv[NF][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int n = min(8, k1 - (k0 + 16 * q + 8 * b));
#pragma unroll
      for (int j = 0; j < NF; ++j) wv[j][b] = load_some(wr[j] + k0 + 8 * b, n);
#pragma unroll
      for (int i = 0; i < MF; ++i) xv[i][b] = load_some(xr[i] + k0 + 8 * b, n);
    }
    wave_whole();
    multiply(xv, wv);
  }
#pragma unroll
  for (int half = 4; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) red[wave - half][i * NF + j][lane] = acc[i][j];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] += red[wave][i * NF + j][lane];
    __syncthreads();
  }
  if (wave != 0) return;
  float* out = p.part + ((int64_t)split * p.P + s.padded) * p.Rp;
#pragma unroll
  for (int i = 0; i < MF; ++i)
    if (i < mf)
#pragma unroll
      for (int j = 0; j < NF; ++j)
        if (16 * j < p.Rp)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = 16 * i + 4 * q + e, r = 16 * j + i16;
            out[(int64_t)n * p.Rp + r] = n < s.rows && r < p.R ? acc[i][j][e] : 0.f;
          }
}

// ---- expand -------------------------------------------------------------------------------------------------------------
// out[row, c] = y[row, c] + s_g sum_r h[row, r] w[group, c, r], h the sum of the splits' parts. A workgroup takes MF x 16
// rows and `cols` columns: h goes to LDS once as [high | low] operands, then every wave takes strips of 64 columns. Of a
// strip, operand row i of fragment j is column 16 (i / 4) + 4 j + i % 4, so a lane's results are 16 consecutive columns of one row.
struct ExpandParams {
  const float* part;
  const uint16_t* w;  // [L, C, ldw], elements beyond R of a row are not read unless wvec (then they are zero)
  int64_t ldw;
  int wvec;           // rows of w are whole 16-byte pieces
  const float* scales;
  const uint16_t* y;  // may be null: zeros
  int64_t ldy;
  uint16_t* out;
  int64_t ldo;
  float* h;           // may be null; [T, R]
  Rows rows;
  int C, R, Rp, P, splits, cols;
};

template <bool F16, int KF, int MF, bool VEC>
__global__ __launch_bounds__(256) void lora_expand(ExpandParams p, int slots) {
  __shared__ __align__(16) uint16_t hs[KF][16 * MF][32];
  __shared__ float row_up[16 * MF];
  __shared__ int row_t[16 * MF];
  const int block = blockIdx.x / slots;
  const Slot s = find_slot(p.rows, blockIdx.x - block * slots, 16 * MF);
  if (s.group < 0) return;
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), i16 = lane & 15, q = lane >> 4;
  const bool none = s.group == p.rows.G - 1;
  const float scale = none ? 0.f : p.scales ? p.scales[s.group] : 1.f;
  const int mf = (s.rows + 15) >> 4;
  if (tid < 16 * MF) {
    const int t = tid < s.rows ? p.rows.perm[s.first + tid] : -1;
    row_t[tid] = t < p.rows.T ? t : -1;
  }
  __syncthreads();
  // four ranks of a row per thread; the KF * 4 threads of a row are neighbours in a wave
  for (int n = tid; n < 16 * MF * KF * 4; n += 256) {
    const int row = n / (KF * 4), r = (n % (KF * 4)) * 4;
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (!none && row < s.rows && r < p.Rp)
      for (int c = 0; c < p.splits; ++c) v += *(const f32x4_t*)(p.part + ((int64_t)c * p.P + s.padded + row) * p.Rp + r);
    if (p.h && block == 0 && row < s.rows && row_t[row] >= 0)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r + e < p.R) p.h[(int64_t)row_t[row] * p.R + r + e] = v[e];
    float f = 1.f, up = scale;
    if (F16) {
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) m = finite_max(m, v[e]);
#pragma unroll
      for (int d = 1; d < KF * 4; d <<= 1) m = max(m, __shfl_xor(m, d, 64));
      f = pow2_down(m);
      up = scale * pow2_up(m);
    }
    if (r == 0) row_up[row] = up;
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint16_t h0, l0, h1, l1;
      split16<F16>(v[2 * e] * f, h0, l0);
      split16<F16>(v[2 * e + 1] * f, h1, l1);
      hi[e] = (uint32_t)h0 | ((uint32_t)h1 << 16);
      lo[e] = (uint32_t)l0 | ((uint32_t)l1 << 16);
    }
    uint16_t* d = &hs[r >> 4][row][r & 15];
    *(u32x2_t*)d = u32x2_t{hi[0], hi[1]};
    *(u32x2_t*)(d + 16) = u32x2_t{lo[0], lo[1]};
  }
  __syncthreads();
  if (none && p.out == p.y) return;

  const int64_t c_begin = (int64_t)block * p.cols;
  const int c_end = (int)min((int64_t)p.C, c_begin + p.cols);
  for (int c0 = (int)c_begin + 64 * wave; c0 < c_end; c0 += 256) {
    // Columns and rows that do not exist read existing ones in their place: their results are not stored.
    u32x4_t wv[KF][4];
#pragma unroll
    for (int k = 0; k < KF; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = min(c0 + 16 * (i16 >> 2) + 4 * j + (i16 & 3), p.C - 1), r = 16 * k + 8 * (q & 1);
        const uint16_t* src = p.w + ((int64_t)s.group * p.C + c) * p.ldw;
        if (none) {
          wv[k][j] = u32x4_t{0u, 0u, 0u, 0u};
        } else if (p.wvec) {
          const u32x4_t v = load16(src + min(r, (int)p.ldw - 8));
          wv[k][j] = r < p.R ? v : u32x4_t{0u, 0u, 0u, 0u};
        } else {
          wv[k][j] = load_some(src + r, p.R - r);
        }
      }
    const int c = c0 + 16 * q;  // this lane's 16 results
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      if (i >= mf) break;
      const int t = row_t[16 * i + i16];
      const float up = row_up[16 * i + i16];
      u32x4_t yv[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        yv[b] = u32x4_t{0u, 0u, 0u, 0u};
        if (p.y) {
          const uint16_t* src = p.y + (int64_t)max(t, 0) * p.ldy;
          yv[b] = VEC ? load16(src + min(c + 8 * b, p.C - 8)) : load_some(src + c + 8 * b, min(8, p.C - c - 8 * b));
        }
      }
      f32x4_t acc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      wave_whole();
#pragma unroll
      for (int k = 0; k < KF; ++k) {
        const u32x4_t hv = *(const u32x4_t*)&hs[k][16 * i + i16][8 * q];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = mfma_16x16x32<F16>(wv[k][j], hv, acc[j]);
      }
      if (t >= 0) {
        uint16_t* dst = p.out + (int64_t)t * p.ldo + c;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          u32x4_t o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // columns 8 b + 2 e and the next one: fragment 2 b + e / 2, results 2 (e % 2) and the next one
            const float v0 = f32_of_16<F16>((uint16_t)(yv[b][e] & 0xFFFFu)), v1 = f32_of_16<F16>((uint16_t)(yv[b][e] >> 16));
            const f32x4_t& a = acc[2 * b + (e >> 1)];
            o[e] = none ? yv[b][e] : pack_16x2<F16>(v0 + up * a[2 * (e & 1)], v1 + up * a[2 * (e & 1) + 1]);
          }
          const int n = min(8, p.C - c - 8 * b);
          if (VEC) {
            if (n > 0) *(u32x4_t*)(dst + 8 * b) = o;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < n) dst[8 * b + e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
          }
        }
      }
      wave_whole();
    }
  }
}

// ---- backward: transposed copies ----------------------------------------------------------------------------------------
// dst[g][c][r] (rows of ldd) = src[g][r][c], for adapters that have rows. Elements between c < Cd's R and ldd are zeros.
__global__ __launch_bounds__(256) void lora_transpose(const uint16_t* src, int Rs, int Cs, uint16_t* dst, int64_t ldd, Rows rows) {
  __shared__ uint16_t tile[64][66];
  const int g = blockIdx.z;
  if (clamp_off(rows, g + 1) <= clamp_off(rows, g)) return;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const uint16_t* s = src + (int64_t)g * Rs * Cs;
  for (int n = threadIdx.x; n < 64 * 64; n += 256) {
    const int r = r0 + (n >> 6), c = c0 + (n & 63);
    tile[n >> 6][n & 63] = r < Rs && c < Cs ? s[(int64_t)r * Cs + c] : (uint16_t)0;
  }
  __syncthreads();
  uint16_t* d = dst + (int64_t)g * Cs * ldd;
  for (int n = threadIdx.x; n < 64 * 64; n += 256) {
    const int c = c0 + (n >> 6), r = r0 + (n & 63);
    if (c < Cs && r < ldd) d[(int64_t)c * ldd + r] = tile[n & 63][n >> 6];
  }
}

// ---- backward: the [rows, R] operand of wgrad ---------------------------------------------------------------------------
// From the splits' parts (or from h as the forward pass returned it, in row order): for rank r and padded row n
// hi[r][n], lo[r][n] = the two 16-bit parts of s_g * value, for fp16 times the power of two that suits the largest of the
// chunk's rows; up[chunk slot][r] is its inverse. A workgroup takes one chunk and four ranks.
struct SmallParams {
  const float* part;
  const float* h;  // instead of part, [T, R]
  const float* scales;
  Rows rows;
  int R, Rp, P, splits, chunk;
  uint16_t* hi;  // [Rp][P]
  uint16_t* lo;
  float* up;     // [chunk slots][Rp]
};

DEVINL float small_value(const SmallParams& p, const Slot& s, int n, int r, float scale) {
  if (n >= s.rows || r >= p.R) return 0.f;
  float v = 0.f;
  if (p.h) {
    const int t = p.rows.perm[s.first + n];
    if (t >= 0 && t < p.rows.T) v = p.h[(int64_t)t * p.R + r];
  } else {
    for (int c = 0; c < p.splits; ++c) v += p.part[((int64_t)c * p.P + s.padded + n) * p.Rp + r];
  }
  return v * scale;
}

template <bool F16>
__global__ __launch_bounds__(256) void lora_small(SmallParams p0, SmallParams p1) {
  __shared__ float wave_max[4][4];
  const SmallParams p = blockIdx.z ? p1 : p0;
  const Slot s = find_slot(p.rows, blockIdx.x, p.chunk);
  if (s.group < 0 || s.group == p.rows.G - 1) return;
  const int tid = threadIdx.x, r = blockIdx.y * 4 + (tid & 3);
  const float scale = p.scales ? p.scales[s.group] : 1.f;
  float f = 1.f;
  if (F16) {
    float m = 0.f;
    for (int n = tid >> 2; n < s.rows; n += 64) m = finite_max(m, small_value(p, s, n, r, scale));
    wave_whole();
#pragma unroll
    for (int d = 4; d < 64; d <<= 1) m = max(m, __shfl_xor(m, d, 64));
    if (lane_id() < 4) wave_max[wave_id()][lane_id()] = m;
    __syncthreads();
    m = max(max(wave_max[0][tid & 3], wave_max[1][tid & 3]), max(wave_max[2][tid & 3], wave_max[3][tid & 3]));
    f = pow2_down(m);
    if (tid < 4) p.up[(int64_t)blockIdx.x * p.Rp + r] = pow2_up(m);
  }
  for (int n = tid >> 2; n < ((s.rows + 15) & ~15); n += 64) {
    uint16_t hi, lo;
    split16<F16>(small_value(p, s, n, r, scale) * f, hi, lo);
    p.hi[(int64_t)r * p.P + s.padded + n] = hi;
    p.lo[(int64_t)r * p.P + s.padded + n] = lo;
  }
}

// ---- backward: wgrad ----------------------------------------------------------------------------------------------------
// grad[c, r] = sum over the rows of an adapter of big[row, c] * small[row, r]. A workgroup takes up to `chunk` rows and 256
// columns, 64 to a wave, in steps of 32 rows: the rows go through LDS as they are and are read back transposed
// (ds_read_b64_tr_b16: four rows of 16 columns per 16 lanes), the small operand is laid out for the matrix instruction already.
// An adapter of one chunk is finished here; the sums of several are added in their order by lora_grad_sum, which also clears
// the gradients of adapters without rows.
struct GradJob {
  const uint16_t* big;
  int64_t ld;
  const uint16_t* hi;
  const uint16_t* lo;
  const float* up;
  uint16_t* grad;  // CR: [L, C, R], else [L, R, C]
  float* part;     // [entries][C * R]
  int C, vec, blocks;
};
struct GradParams {
  GradJob job[2];  // gB (as [C, R]), gA (as [R, C])
  Rows rows;
  int R, Rp, P, chunk, slots, vec_store;  // vec_store: four neighbours of a gradient can be stored together
};

constexpr int GRAD_ROW = 272;   // elements from row to row in LDS (256 columns and 32 bytes to spread the banks)
constexpr int GRAD_SKEW = 64;   // and after every eight rows
DEVINL int grad_off(int row) { return row * GRAD_ROW + (row >> 3) * GRAD_SKEW; }
constexpr int GRAD_TILE = 32 * GRAD_ROW + 4 * GRAD_SKEW;

DEVINL u32x4_t read_transposed(const uint16_t* at) {
  typedef __attribute__((address_space(3))) i16x4_t* lds_ptr;
  const uint32_t a = (uint32_t)(uintptr_t)at;
  const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)a);
  const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(a + 4 * GRAD_ROW * 2));
  const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
  return u32x4_t{l2[0], l2[1], h2[0], h2[1]};
}

template <bool F16, int RF, bool CR>
DEVINL void grad_body(const GradParams& p, const GradJob& job, int block, int slot, uint16_t* tile, uint16_t* small) {
  const Slot s = find_slot(p.rows, slot, p.chunk);
  if (s.group < 0 || s.group == p.rows.G - 1) return;
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), i16 = lane & 15, q = lane >> 4;
  const int c0 = block * 256, rows16 = (s.rows + 15) & ~15;
  f32x4_t acc[4][RF];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int f = 0; f < RF; ++f) acc[j][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  constexpr int SMALL = 2 * RF * 16 * 4;        // 16-byte pieces of the small operand per step
  constexpr int SL = (SMALL + 255) / 256;
  u32x4_t bv[4], sv[SL];
  auto load = [&](int n0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + (tid >> 5) + 8 * j, c = c0 + 8 * (tid & 31);
      const int t = n < s.rows ? p.rows.perm[s.first + n] : -1;
      const int some = t >= 0 && t < p.rows.T ? min(8, job.C - c) : 0;
      bv[j] = u32x4_t{0u, 0u, 0u, 0u};
      if (some > 0) {
        const uint16_t* src = job.big + (int64_t)t * job.ld + c;
        bv[j] = job.vec ? load16(src) : load_some(src, some);
      }
    }
#pragma unroll
    for (int j = 0; j < SL; ++j) {
      const int i = tid + 256 * j, n = n0 + 8 * (i & 3), r = (i >> 2) % (RF * 16);
      sv[j] = u32x4_t{0u, 0u, 0u, 0u};
      if (i < SMALL && n < rows16 && r < p.Rp) sv[j] = load16((i >= SMALL / 2 ? job.lo : job.hi) + (int64_t)r * p.P + s.padded + n);
    }
  };
  load(0);
  int buf = 0;
  for (int n0 = 0; n0 < s.rows; n0 += 32, buf ^= 1) {
    uint16_t* tl = tile + buf * GRAD_TILE;
    uint16_t* sm = small + buf * (SMALL * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) *(u32x4_t*)(tl + grad_off((tid >> 5) + 8 * j) + 8 * (tid & 31)) = bv[j];
#pragma unroll
    for (int j = 0; j < SL; ++j)
      if (tid + 256 * j < SMALL) *(u32x4_t*)(sm + (tid + 256 * j) * 8) = sv[j];
    if (n0 + 32 < s.rows) load(n0 + 32);
    __syncthreads();
    u32x4_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = read_transposed(tl + grad_off(8 * q + (i16 >> 2)) + 64 * wave + 16 * j + 4 * (i16 & 3));
#pragma unroll
    for (int f = 0; f < RF; ++f)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4_t v = *(const u32x4_t*)(sm + ((h * RF * 16 + 16 * f + i16) * 4 + q) * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][f] = CR ? mfma_16x16x32<F16>(v, b[j], acc[j][f]) : mfma_16x16x32<F16>(b[j], v, acc[j][f]);
      }
  }
  const bool whole = s.size <= p.chunk;
  const int64_t block_size = (int64_t)job.C * p.R;
  const int64_t entry = s.begin / (p.chunk / 2) + (s.first - s.begin) / p.chunk;
  uint16_t* grad = job.grad + s.group * block_size;
  float* part = job.part + entry * block_size;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      const int c = c0 + 64 * wave + 16 * j + (CR ? i16 : 4 * q), r = 16 * f + (CR ? 4 * q : i16);
      if (c >= job.C || r >= p.R) continue;
      f32x4_t v = acc[j][f];
      if (F16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= job.up[(int64_t)slot * p.Rp + r + (CR ? e : 0)];
      }
      const int64_t at = CR ? (int64_t)c * p.R + r : (int64_t)r * job.C + c;
      const int n = min(4, CR ? p.R - r : job.C - c);
      if (p.vec_store) {
        if (whole) *(u32x2_t*)(grad + at) = u32x2_t{pack_16x2<F16>(v[0], v[1]), pack_16x2<F16>(v[2], v[3])};
        else *(f32x4_t*)(part + at) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < n) {
            if (whole) grad[at + e] = cvt_16<F16>(v[e]);
            else part[at + e] = v[e];
          }
      }
    }
}

template <bool F16, int RF>
__global__ __launch_bounds__(256) void lora_grad(GradParams p) {
  __shared__ __align__(16) uint16_t tile[2 * GRAD_TILE];
  __shared__ __align__(16) uint16_t small[2 * 2 * RF * 16 * 32];
  const int slot = blockIdx.x % p.slots, block = blockIdx.x / p.slots;
  if (block < p.job[0].blocks) grad_body<F16, RF, true>(p, p.job[0], block, slot, tile, small);
  else grad_body<F16, RF, false>(p, p.job[1], block - p.job[0].blocks, slot, tile, small);
}

template <bool F16>
__global__ __launch_bounds__(256) void lora_grad_sum(GradParams p, int blocks0) {
  const int g = blockIdx.y;
  const int begin = clamp_off(p.rows, g), size = clamp_off(p.rows, g + 1) - begin;
  if (size > 0 && size <= p.chunk) return;
  const bool first = (int)blockIdx.x < blocks0;
  const GradJob& job = first ? p.job[0] : p.job[1];
  const int64_t block_size = (int64_t)job.C * p.R;
  const int64_t i = ((int64_t)(blockIdx.x - (first ? 0 : blocks0)) * 256 + threadIdx.x) * 4;
  if (i >= block_size) return;
  const int n = (int)min((int64_t)4, block_size - i);
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const int chunks = size > 0 ? (size + p.chunk - 1) / p.chunk : 0;
  for (int c = 0; c < chunks; ++c) {
    const float* part = job.part + ((int64_t)(begin / (p.chunk / 2)) + c) * block_size + i;
    for (int e = 0; e < n; ++e) v[e] += part[e];
  }
  uint16_t* d = job.grad + g * block_size + i;
  for (int e = 0; e < n; ++e) d[e] = cvt_16<F16>(v[e]);
}

template <bool F16, int NF, int MF>
void launch_shrink(const ShrinkParams& p, bool vec, hipStream_t stream) {
  const int slots = p.rows.T / (16 * MF) + p.rows.G;
  const dim3 grid(slots * p.splits), block(512);
  if (vec) hipLaunchKernelGGL((lora_shrink<F16, NF, MF, true>), grid, block, 0, stream, p, slots);
  else hipLaunchKernelGGL((lora_shrink<F16, NF, MF, false>), grid, block, 0, stream, p, slots);
}

template <bool F16, int KF, int MF>
void launch_expand(const ExpandParams& p, bool vec, hipStream_t stream) {
  const int slots = p.rows.T / (16 * MF) + p.rows.G;
  const dim3 grid(slots * ((p.C + p.cols - 1) / p.cols)), block(256);
  if (vec) hipLaunchKernelGGL((lora_expand<F16, KF, MF, true>), grid, block, 0, stream, p, slots);
  else hipLaunchKernelGGL((lora_expand<F16, KF, MF, false>), grid, block, 0, stream, p, slots);
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
int rank_blocks(int R) { return R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8; }
// Rows per workgroup of shrink and expand: 64 (32 for the highest ranks in shrink) reuse an adapter's weights over more
// rows, 16 give more workgroups; below 512 rows there are too few of the former to fill the card.
constexpr int MANY_ROWS = 512;

template <bool F16>
void shrink(const ShrinkParams& p, hipStream_t stream) {
  const bool vec = p.C % 8 == 0 && p.ldx % 8 == 0 && p.ldw % 8 == 0 && aligned16(p.x) && aligned16(p.w);
  const bool many = p.rows.T >= MANY_ROWS;
  switch (rank_blocks(p.R)) {
    case 1: many ? launch_shrink<F16, 1, 4>(p, vec, stream) : launch_shrink<F16, 1, 1>(p, vec, stream); break;
    case 2: many ? launch_shrink<F16, 2, 4>(p, vec, stream) : launch_shrink<F16, 2, 1>(p, vec, stream); break;
    case 4: many ? launch_shrink<F16, 4, 4>(p, vec, stream) : launch_shrink<F16, 4, 1>(p, vec, stream); break;
    default: many ? launch_shrink<F16, 8, 2>(p, vec, stream) : launch_shrink<F16, 8, 1>(p, vec, stream); break;
  }
}

template <bool F16>
void expand(const ExpandParams& p, hipStream_t stream) {
  const bool vec = p.C % 8 == 0 && p.ldy % 8 == 0 && p.ldo % 8 == 0 && aligned16(p.y) && aligned16(p.out);
  const bool many = p.rows.T >= MANY_ROWS;
  switch (rank_blocks(p.R)) {
    case 1: many ? launch_expand<F16, 1, 4>(p, vec, stream) : launch_expand<F16, 1, 1>(p, vec, stream); break;
    case 2: many ? launch_expand<F16, 2, 4>(p, vec, stream) : launch_expand<F16, 2, 1>(p, vec, stream); break;
    case 4: many ? launch_expand<F16, 4, 4>(p, vec, stream) : launch_expand<F16, 4, 1>(p, vec, stream); break;
    default: many ? launch_expand<F16, 8, 4>(p, vec, stream) : launch_expand<F16, 8, 1>(p, vec, stream); break;
  }
}

// Splits of the reduced axis: until about 512 workgroups (two to a CU), but 64 columns at least for each of the eight waves
// and at most 16 parts, which the next kernel adds again for every row.
int shrink_splits(int64_t T, int G, int R, int C) {
  const int64_t rows = T >= MANY_ROWS ? (rank_blocks(R) == 8 ? 32 : 64) : 16;
  const int64_t tiles = T / rows + (G < T ? G : T) + (T == 0);
  const int64_t most = (C + 511) / 512;
  int64_t s = 512 / tiles;
  s = s < 1 ? 1 : s > 16 ? 16 : s;
  return (int)(s < most ? s : most);
}
int per_wave(int C, int splits) { return (int)((((int64_t)C + 64 * 8 * splits - 1) / (64 * 8 * splits)) * 64); }

struct Sizes {
  int64_t G, P, Rp, chunk, slots, entries;
  int s_x, s_g;
};
Sizes sizes_of(int64_t T, int L, int K, int N, int R) {
  Sizes z;
  z.G = L + 1;
  z.P = 16 * (T / 16 + z.G);
  z.Rp = (R + 15) / 16 * 16;
  z.chunk = 512 * (T > 8192 ? (T + 8191) / 8192 : 1);
  z.slots = T / z.chunk + z.G;
  z.entries = T / (z.chunk / 2);
  z.s_x = shrink_splits(T, (int)z.G, R, K);
  z.s_g = shrink_splits(T, (int)z.G, R, N);
  return z;
}

struct Workspace {
  char* base;
  size_t used;
  template <class V> V* take(int64_t n) {
    V* p = (V*)(base + used);
    used += ((size_t)n * sizeof(V) + 255) / 256 * 256;
    return p;
  }
};

struct BackwardSpace {
  uint16_t *bt, *at, *hi[2], *lo[2];
  float *part_u, *part_h, *up[2], *sums[2];
};
BackwardSpace backward_space(Workspace& w, const Sizes& z, int L, int K, int N, int R, bool with_h) {
  BackwardSpace b;
  b.bt = w.take<uint16_t>((int64_t)L * R * ((N + 7) / 8 * 8));
  b.at = w.take<uint16_t>((int64_t)L * K * ((R + 7) / 8 * 8));
  b.part_u = w.take<float>(z.s_g * z.P * z.Rp);
  b.part_h = with_h ? nullptr : w.take<float>(z.s_x * z.P * z.Rp);
  for (int j = 0; j < 2; ++j) {
    b.hi[j] = w.take<uint16_t>(z.Rp * z.P);
    b.lo[j] = w.take<uint16_t>(z.Rp * z.P);
    b.up[j] = w.take<float>(z.slots * z.Rp);
  }
  b.sums[0] = w.take<float>(z.entries * N * R);
  b.sums[1] = w.take<float>(z.entries * K * R);
  return b;
}

// ids outside [0, L) become L, the group of rows without an adapter.
__global__ __launch_bounds__(256) void lora_keys(const int32_t* ids, int32_t* keys, int T, int L) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < T) keys[t] = ids[t] >= 0 && ids[t] < L ? ids[t] : L;
}

ShrinkParams shrink_params(const void* x, int64_t ldx, const void* w, int64_t ldw, float* part, const Rows& rows, int C, int R, const Sizes& z, int splits) {
  ShrinkParams p{};
  p.x = (const uint16_t*)x; p.ldx = ldx; p.w = (const uint16_t*)w; p.ldw = ldw; p.part = part; p.rows = rows;
  p.C = C; p.R = R; p.Rp = (int)z.Rp; p.P = (int)z.P; p.splits = splits; p.per_wave = per_wave(C, splits);
  return p;
}

// Columns per workgroup of expand: 1024 (four strips per wave) once that fills the card, else 256.
int expand_cols(int64_t T, int G, int C) {
  const int64_t rows = T >= MANY_ROWS ? 64 : 16;
  const int64_t tiles = T / rows + (G < T ? G : T);
  return tiles * ((C + 1023) / 1024) >= 512 ? 1024 : 256;
}

template <bool F16>
void forward(const LoraParams& p, hipStream_t stream) {
  const Sizes z = sizes_of(p.T, p.L, p.K, p.N, p.R);
  const Rows rows{p.perm, p.offsets, (int)z.G, p.T};
  float* part = (float*)p.workspace;
  if (p.L > 0) shrink<F16>(shrink_params(p.x, p.ldx, p.a, p.K, part, rows, p.K, p.R, z, z.s_x), stream);
  ExpandParams e{};
  e.part = part; e.w = (const uint16_t*)p.b; e.ldw = p.R; e.wvec = p.R % 8 == 0 && aligned16(p.b); e.scales = p.scales;
  e.y = (const uint16_t*)p.y; e.ldy = p.ldy; e.out = (uint16_t*)p.out; e.ldo = p.ldo; e.h = (float*)p.h; e.rows = rows;
  e.C = p.N; e.R = p.R; e.Rp = (int)z.Rp; e.P = (int)z.P; e.splits = z.s_x; e.cols = expand_cols(p.T, (int)z.G, p.N);
  expand<F16>(e, stream);
}

template <bool F16, int RF>
void launch_grad(const GradParams& g, hipStream_t stream) {
  hipLaunchKernelGGL((lora_grad<F16, RF>), dim3(g.slots * (g.job[0].blocks + g.job[1].blocks)), dim3(256), 0, stream, g);
}

template <bool F16>
void backward(const LoraParams& p, hipStream_t stream) {
  const Sizes z = sizes_of(p.T, p.L, p.K, p.N, p.R);
  Workspace w{(char*)p.workspace, 0};
  const BackwardSpace b = backward_space(w, z, p.L, p.K, p.N, p.R, p.h != nullptr);
  const Rows rows{p.perm, p.offsets, (int)z.G, p.T};
  const int Nd = (p.N + 7) / 8 * 8, Rd = (p.R + 7) / 8 * 8;
  ExpandParams e{};
  e.part = b.part_u; e.w = b.at; e.ldw = Rd; e.wvec = 1; e.scales = p.scales; e.y = (const uint16_t*)p.gx_in; e.ldy = p.ld_gx_in;
  e.out = (uint16_t*)p.gx; e.ldo = p.ld_gx; e.rows = rows; e.C = p.K; e.R = p.R; e.Rp = (int)z.Rp; e.P = (int)z.P; e.splits = z.s_g;
  e.cols = expand_cols(p.T, (int)z.G, p.K);
  if (!e.y) e.ldy = e.ldo;
  if (p.L == 0) return expand<F16>(e, stream);
  hipLaunchKernelGGL(lora_transpose, dim3((p.R + 63) / 64, (Nd + 63) / 64, p.L), dim3(256), 0, stream, (const uint16_t*)p.b, p.N, p.R, b.bt, (int64_t)Nd, rows);
  hipLaunchKernelGGL(lora_transpose, dim3((p.K + 63) / 64, (Rd + 63) / 64, p.L), dim3(256), 0, stream, (const uint16_t*)p.a, p.R, p.K, b.at, (int64_t)Rd, rows);
  shrink<F16>(shrink_params(p.y, p.ldy, b.bt, Nd, b.part_u, rows, p.N, p.R, z, z.s_g), stream);
  if (!p.h) shrink<F16>(shrink_params(p.x, p.ldx, p.a, p.K, b.part_h, rows, p.K, p.R, z, z.s_x), stream);
  SmallParams sp[2] = {};
  for (int j = 0; j < 2; ++j) {  // 0: h for gB, 1: u for gA
    sp[j].part = j ? b.part_u : b.part_h;
    sp[j].h = j ? nullptr : (const float*)p.h;
    sp[j].scales = p.scales; sp[j].rows = rows; sp[j].R = p.R; sp[j].Rp = (int)z.Rp; sp[j].P = (int)z.P;
    sp[j].splits = j ? z.s_g : z.s_x; sp[j].chunk = (int)z.chunk; sp[j].hi = b.hi[j]; sp[j].lo = b.lo[j]; sp[j].up = b.up[j];
  }
  hipLaunchKernelGGL((lora_small<F16>), dim3((unsigned)z.slots, (unsigned)z.Rp / 4, 2), dim3(256), 0, stream, sp[0], sp[1]);
  expand<F16>(e, stream);
  GradParams g{};
  g.rows = rows; g.R = p.R; g.Rp = (int)z.Rp; g.P = (int)z.P; g.chunk = (int)z.chunk; g.slots = (int)z.slots;
  g.vec_store = p.R % 4 == 0 && p.K % 4 == 0 && (uintptr_t)p.grad_a % 8 == 0 && (uintptr_t)p.grad_b % 8 == 0;
  for (int j = 0; j < 2; ++j) {
    GradJob& job = g.job[j];
    job.big = (const uint16_t*)(j ? p.x : p.y);
    job.ld = j ? p.ldx : p.ldy;
    job.hi = b.hi[j]; job.lo = b.lo[j]; job.up = b.up[j];
    job.grad = (uint16_t*)(j ? p.grad_a : p.grad_b);
    job.part = b.sums[j];
    job.C = j ? p.K : p.N;
    job.vec = job.C % 8 == 0 && job.ld % 8 == 0 && aligned16(job.big);
    job.blocks = (job.C + 255) / 256;
  }
  switch (rank_blocks(p.R)) {
    case 1: launch_grad<F16, 1>(g, stream); break;
    case 2: launch_grad<F16, 2>(g, stream); break;
    case 4: launch_grad<F16, 4>(g, stream); break;
    default: launch_grad<F16, 8>(g, stream); break;
  }
  const int blocks0 = (int)(((int64_t)p.N * p.R + 1023) / 1024), blocks1 = (int)(((int64_t)p.K * p.R + 1023) / 1024);
  hipLaunchKernelGGL((lora_grad_sum<F16>), dim3(blocks0 + blocks1, p.L), dim3(256), 0, stream, g, blocks0);
}

}  // namespace

size_t lora_forward_workspace(int64_t T, int L, int K, int N, int R) {
  const Sizes z = sizes_of(T, L, K, N, R);
  return (size_t)z.s_x * z.P * z.Rp * sizeof(float);
}

size_t lora_backward_workspace(int64_t T, int L, int K, int N, int R, bool with_h) {
  Workspace w{nullptr, 0};
  backward_space(w, sizes_of(T, L, K, N, R), L, K, N, R, with_h);
  return w.used;
}

hipError_t lora_plan_launch(const int32_t* ids, int T, int L, int32_t* perm, int32_t* offsets, int32_t* scratch, hipStream_t stream) {
  if (T > 0) hipLaunchKernelGGL(lora_keys, dim3((T + 255) / 256), dim3(256), 0, stream, ids, scratch, T, L);
  return route_group_launch(scratch, T, L + 1, perm, scratch + T, offsets, stream);
}

hipError_t lora_forward_launch(const LoraParams& p, bool fp16, hipStream_t stream) {
  fp16 ? forward<true>(p, stream) : forward<false>(p, stream);
  return hipGetLastError();
}

hipError_t lora_backward_launch(const LoraParams& p, bool fp16, hipStream_t stream) {
  fp16 ? backward<true>(p, stream) : backward<false>(p, stream);
  return hipGetLastError();
}
