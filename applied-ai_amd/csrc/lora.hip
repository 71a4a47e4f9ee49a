// Low-rank adapters of many requests beside one shared projection, and their gradients.
//
// Row t of a batch names an adapter e = id(t) with matrices A_e [R, K] and B_e [N, R] and a factor s_e:
//   h[t] = A_e x[t]                     out[t] = y[t] + s_e B_e h[t]                 (rows without an adapter: out = y)
//   u[t] = s_e B_e^T gout[t]            gx[t] = gx_in[t] + A_e^T u[t]
//   gA_e = sum_t u[t] x[t]^T            gB_e = s_e sum_t gout[t] h[t]^T
// The rank R is small, so every product moves far more bytes than it computes: x, y, out, gout, gx pass through the kernels and
// the matrix instructions only keep up with memory. Three kernels do all of it:
//   shrink  [rows, C] . [R, C]^T  -> [rows, R]   the long axis C is reduced: split over workgroups and waves
//   expand  [rows, R] . [C, R]^T  -> [rows, C]   added to a row of y on its way through
//   wgrad   [rows, C]^T . [rows, R] -> [C, R]    rows are reduced, adapter by adapter; on the output's gradient it also takes
//                                                the product with B (u) from the same rows, which are then read once
// and for a few rows shrink and expand are one kernel without an intermediate in memory.
//
// Rows are taken in adapter order (perm, offsets of the plan). Group g = adapter g for g < L and "no adapter" for g = L.
// A grid cannot know the groups' sizes without a copy to the host, so it counts slots of `unit` rows:
// group g owns slots [off_g / unit + g, off_{g+1} / unit + g + 1), at least as many as it needs, and a workgroup
// finds its group with one ballot over the group table (two beyond 64 groups). [rows, R] intermediates live in the same space
// with unit 16: group g's rows start at 16 * (off_g / 16 + g), so that every group is aligned and padded with zero rows.
//
// Where that is fewer, slots are the rows themselves, of which every unit-th of a group has work (a few single tokens beside
// many loaded adapters).
//
// The intermediates are fp32. As matrix operands they are split into parts of the 16-bit type, each the rounding of what the parts
// before it leave: three of bf16, which hold all 24 bits, or two of fp16, which hold 22 (a result in fp16 has 11). One matrix
// instruction covers two parts of 16 ranks, its 32-deep reduction holding [first 16 | second 16] against the same 16 columns of
// the other operand twice; the third part takes another one. Two parts of bf16 would be off by 2^-17, many times the error of the
// fp32 sums around them. The third costs nothing at rank 16 (4096 rows of 4096 -> 14336: expand 58 us with and without it, the
// gradients' kernels 44 + 14 us) and 5 to 16 % of a kernel from rank 64 on, where the matrix instructions count (rank 128: expand
// 318 -> 341 us, the gradients' 203 -> 217 and 45 -> 46 us). For fp16 the rows are scaled by a power of two first, so that
// neither part leaves the type's range.
#include "common.h"
#include "kernels.h"

namespace {

typedef short i16x4_t __attribute__((ext_vector_type(4)));

template <int N> struct Number { static constexpr int value = N; };

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
  int of;      // the group that owns the slot, also where it holds nothing
};

DEVINL Slot slot_of(bool by_row, int v, int unit, int g, int begin, int end) {
  int skip = (v - (begin / unit + g)) * unit;
  if (by_row) skip = (v - begin) % unit == 0 ? v - begin : -1;
  Slot s;
  s.begin = begin;
  s.size = end - begin;
  s.first = begin + skip;
  s.rows = min(unit, s.size - skip);
  s.padded = 16 * (begin / 16 + g) + skip;
  s.group = s.rows > 0 && skip >= 0 ? g : -1;
  s.of = g;
  return s;
}
// Which rows slot v of `unit` rows holds. All lanes of the wave take part; the result is the same in all of them. Whatever
// the table holds, the rows named lie inside [0, T).
DEVINL Slot find_slot(const Rows& r, int v, int unit, bool by_row) {
  const int lane = lane_id();
  if (r.G < 64) {  // the whole table in one load
    const int off = clamp_off(r, min(lane, r.G));
    const int g = min(max(__popcll(__ballot(lane < r.G && (by_row ? off : off / unit + lane) <= v)) - 1, 0), r.G - 1);
    return slot_of(by_row, v, unit, g, __shfl(off, g, 64), __shfl(off, g + 1, 64));
  }
  const int step = (r.G + 63) >> 6;
  int i = lane * step;
  int off = clamp_off(r, min(i, r.G));
  bool le = i < r.G && (by_row ? off : off / unit + i) <= v;
  int g = max(__popcll(__ballot(le)) - 1, 0) * step;
  if (step > 1) {
    i = g + lane;
    off = clamp_off(r, min(i, r.G));
    le = lane < step && i < r.G && (by_row ? off : off / unit + i) <= v;
    g += max(__popcll(__ballot(le)) - 1, 0);
  }
  g = min(g, r.G - 1);
  return slot_of(by_row, v, unit, g, clamp_off(r, g), clamp_off(r, g + 1));
}
DEVINL Slot find_slot(const Rows& r, int v, int unit) { return find_slot(r, v, unit, r.T < r.T / unit + r.G); }

// Eight elements at any address: the hardware's wide loads and stores need no alignment, and what an unaligned one costs
// is the second line that it may touch.
typedef u32x4_t u32x4_any_t __attribute__((aligned(2)));
typedef u32x2_t u32x2_any_t __attribute__((aligned(2)));
typedef f32x4_t f32x4_any_t __attribute__((aligned(4)));
DEVINL u32x4_t load16(const uint16_t* p) { return *(const u32x4_any_t*)p; }
DEVINL void store16(uint16_t* p, u32x4_t v) { *(u32x4_any_t*)p = v; }
// Eight elements p[0..7] of which only the first n exist (none for n <= 0), with `before` elements in front of p: from the
// eight that end with the last one where there are as many.
DEVINL u32x4_t load_some(const uint16_t* p, int n, int before) {
  u32x4_t v = {0u, 0u, 0u, 0u};
  if (n > 0 && n + before >= 8) {
    const u32x4_t w = load16(p - (8 - n));
    const uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
    const int s = 16 * (8 - n);  // 16 .. 112
    const uint64_t a = s < 64 ? lo >> (s & 63) | hi << ((64 - s) & 63) : hi >> ((s - 64) & 63), b = s < 64 ? hi >> (s & 63) : 0;
    return u32x4_t{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)};
  }
#pragma unroll
  for (int e = 0; e < 7; ++e)
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
template <bool F16> constexpr int PARTS = F16 ? 2 : 3;
// v as a sum of parts of the 16-bit type; of an infinity or NaN the first one is all.
template <bool F16> DEVINL void split16(float v, uint16_t (&part)[PARTS<F16>]) {
  part[0] = cvt_16<F16>(v);
  float r = v - f32_of_16<F16>(part[0]);
  if (!(__builtin_fabsf(r) <= 3.4028234e38f)) r = 0.f;
#pragma unroll
  for (int i = 1; i < PARTS<F16>; ++i) {
    part[i] = cvt_16<F16>(r);
    r -= f32_of_16<F16>(part[i]);
  }
}

// ---- shrink -------------------------------------------------------------------------------------------------------------
// part[split][padded row][r] = sum over the split's columns of x[row, c] * w[group, r, c].
// A workgroup takes MF x 16 rows and one split; its eight waves take an eighth of the split each and are summed through LDS.
// A row is read by four lanes, 64 consecutive bytes at a time. Bound by the latency of its chain of loads (group table, rows, columns)
// and by HBM: 4096 x 4096 bf16, rank 16, 14 us (2.4 TB/s); 64 rows of 14336 and 32 adapters 8 us.
struct ShrinkParams {
  const uint16_t* x;
  int64_t ldx;
  const uint16_t* w;  // [L, R, ldw]
  int64_t ldw;
  float* part;        // [S][P][Rp]
  Rows rows;
  int C, R, Rp, P, splits, per_wave;  // per_wave: columns per wave, a multiple of 64
};

// acc += the products of columns [k0, k1) of a wave: xr, wr point at column 8 q of this lane's rows, MANY x 64 columns have
// their loads under way before the first product.
template <bool F16, int NF, int MF, int MANY>
DEVINL void shrink_columns(const uint16_t* const (&xr)[MF], const uint16_t* const (&wr)[NF], int k0, int k1, int q, f32x4_t (&acc)[MF][NF]) {
  auto columns = [&](int k, auto steps) {
    constexpr int STEPS = decltype(steps)::value;
    u32x4_t xv[STEPS][2][MF], wv[STEPS][2][NF];
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int i = 0; i < MF; ++i) xv[s][b][i] = load16(xr[i] + k + 64 * s + 32 * b);
#pragma unroll
        for (int j = 0; j < NF; ++j) wv[s][b][j] = load16(wr[j] + k + 64 * s + 32 * b);
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
          for (int j = 0; j < NF; ++j) acc[i][j] = mfma_16x16x32<F16>(xv[s][b][i], wv[s][b][j], acc[i][j]);
  };
  for (; k0 + 64 * MANY <= k1; k0 += 64 * MANY) columns(k0, Number<MANY>());
  if (MANY > 1)
    for (; k0 + 64 <= k1; k0 += 64) columns(k0, Number<1>());
  if (k0 < k1) {  // the last columns of a width that is no multiple of 64
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int n = k1 - (k0 + 8 * q + 32 * b);
      u32x4_t xv[MF], wv[NF];
#pragma unroll
      for (int i = 0; i < MF; ++i) xv[i] = n >= 8 ? load16(xr[i] + k0 + 32 * b) : load_some(xr[i] + k0 + 32 * b, n, k0 + 8 * q + 32 * b);
#pragma unroll
      for (int j = 0; j < NF; ++j) wv[j] = n >= 8 ? load16(wr[j] + k0 + 32 * b) : load_some(wr[j] + k0 + 32 * b, n, k0 + 8 * q + 32 * b);
      wave_whole();
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = mfma_16x16x32<F16>(xv[i], wv[j], acc[i][j]);
    }
  }
}

// The operand rows of a lane. Rows that do not exist read an existing one in their place: a result belongs to one row of
// each operand, and theirs are not kept.
template <int MF> DEVINL void shrink_rows(const Rows& rows, const Slot& s, const uint16_t* x, int64_t ldx, const uint16_t* (&xr)[MF]) {
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int t = rows.perm[s.first + min(16 * i + (lane_id() & 15), s.rows - 1)];
    xr[i] = x + (int64_t)(t >= 0 && t < rows.T ? t : 0) * ldx + 8 * (lane_id() >> 4);
  }
}
template <int NF> DEVINL void shrink_weights(const Slot& s, const uint16_t* w, int64_t ldw, int R, const uint16_t* (&wr)[NF]) {
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int r = 16 * j + (lane_id() & 15);
    wr[j] = w + ((int64_t)s.group * R + (r < R ? r : 0)) * ldw + 8 * (lane_id() >> 4);
  }
}

template <bool F16, int NF, int MF>
__global__ __launch_bounds__(512) void lora_shrink(ShrinkParams p, int slots) {
  constexpr int WAVES = MF * NF > 8 ? 4 : 8;  // whose sums are in LDS at a time: 64 KB at most
  __shared__ __align__(16) float red[WAVES][16 * MF][16 * NF];
  const int split = blockIdx.x / slots;
  const Slot s = find_slot(p.rows, blockIdx.x - split * slots, 16 * MF);
  if (s.group < 0 || s.group == p.rows.G - 1) return;
  const int lane = lane_id(), wave = wave_id(), i16 = lane & 15, q = lane >> 4;
  const uint16_t* xr[MF];
  const uint16_t* wr[NF];
  shrink_rows<MF>(p.rows, s, p.x, p.ldx, xr);
  shrink_weights<NF>(s, p.w, p.ldw, p.R, wr);
  f32x4_t acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int64_t begin = (int64_t)(split * 8 + wave) * p.per_wave;
  shrink_columns<F16, NF, MF, (MF + NF <= 2 ? 2 : 1)>(xr, wr, (int)min(begin, (int64_t)p.C), (int)min((int64_t)p.C, begin + p.per_wave), q, acc);
  auto put = [&](int w) {
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[w][16 * i + 4 * q + e][16 * j + i16] = acc[i][j][e];
  };
  if (WAVES == 4) {
    if (wave >= 4) put(wave - 4);
    __syncthreads();
    if (wave < 4)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += red[wave][16 * i + 4 * q + e][16 * j + i16];
  }
  if (wave < WAVES) put(wave);
  __syncthreads();
  float* out = p.part + ((int64_t)split * p.P + s.padded) * p.Rp;
  for (int n = threadIdx.x; n < 64 * MF * NF; n += 512) {  // four ranks of a row
    const int row = n / (4 * NF), r = 4 * (n % (4 * NF));
    if (row >= ((s.rows + 15) & ~15) || r >= p.Rp) continue;
    f32x4_t v = *(const f32x4_t*)&red[0][row][r];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += *(const f32x4_t*)&red[w][row][r];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row >= s.rows || r + e >= p.R) v[e] = 0.f;
    *(f32x4_t*)(out + (int64_t)row * p.Rp + r) = v;
  }
}

// ---- expand -------------------------------------------------------------------------------------------------------------
// out[row, c] = y[row, c] + s_g sum_r h[row, r] w[group, c, r], h the sum of the splits' parts. A workgroup takes MF x 16
// rows and `cols` columns: h goes to LDS once in its parts, every wave takes strips of 64 columns. Of a
// strip, operand row i of fragment j is column 32 (j / 2) + 8 (i / 4) + 4 (j % 2) + i % 4: a lane's results are twice eight
// consecutive columns of one row, and the four lanes of a row store 64 consecutive bytes.
// WT: w is [group, r, c] (the backward pass with A): a strip of it goes through the wave's LDS and is read back transposed.
// Bound by HBM: 4096 rows of 14336 bf16 read and written in 58 us (4.0 TB/s; a copy reaches 4.9); non-temporal stores take 68 us.
// Higher ranks hold more of w in registers: 90, 109 and 341 us at rank 32, 64 and 128, with three, two and one waves to a SIMD.
struct ExpandParams {
  const float* part;
  const uint16_t* w;  // [L, C, R], WT: [L, R, C]
  const float* scales;
  const uint16_t* y;  // may be null: zeros
  int64_t ldy;
  uint16_t* out;
  int64_t ldo;
  float* h;           // may be null; [T, R]
  Rows rows;
  int C, R, Rp, P, splits, cols;
};

// Four rows of 16 columns per 16 lanes, read transposed from LDS: lane i gets column i of rows 0..3 at `at` and of the four
// rows `next` bytes on. A lane's address is row (i / 4)'s, four columns at (i % 4)'s place.
DEVINL u32x4_t read_transposed(const uint16_t* at, uint32_t next) {
  typedef __attribute__((address_space(3))) i16x4_t* lds_ptr;
  const uint32_t a = (uint32_t)(uintptr_t)at;
  const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)a);
  const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(a + next));
  const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
  return u32x4_t{l2[0], l2[1], h2[0], h2[1]};
}

// The rows of a lane (operand column i16 of each fragment), -1 where there is none.
template <int MF> DEVINL void lane_rows(const Rows& rows, const Slot& s, int (&t)[MF]) {
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int n = 16 * i + (lane_id() & 15);
    t[i] = n < s.rows ? rows.perm[s.first + n] : -1;
    if (t[i] >= rows.T) t[i] = -1;
  }
}

// The parts of a workgroup's rows of h, as the matrix instructions take them.
template <bool F16, int KF, int MF> struct Parts {
  uint16_t pair[KF][16 * MF][32];                        // first and second part of 16 ranks
  uint16_t third[F16 ? 1 : KF][F16 ? 1 : 16 * MF][16];
};

constexpr int WT_ROW = 72;  // elements from rank to rank of a transposed strip in LDS

// A strip of 64 columns of a wave: what it reads, and what it makes of it.
template <bool F16, int KF, int MF, bool WT>
struct Strip {
  u32x4_t y[MF][2], w[KF][4];

  // EDGE: the strip reaches beyond the last column (a case of its own, to keep what every strip runs through short)
  DEVINL void load(const ExpandParams& p, int group, bool none, const int (&t)[MF], int c0) {
    if (c0 + 64 <= p.C) load<false>(p, group, none, t, c0);
    else load<true>(p, group, none, t, c0);
  }
  // rows and columns that do not exist read existing ones: their results are not stored
  template <bool EDGE> DEVINL void load(const ExpandParams& p, int group, bool none, const int (&t)[MF], int c0) {
    const int i16 = lane_id() & 15, q = lane_id() >> 4, c = c0 + 8 * q;
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b) y[i][b] = u32x4_t{0u, 0u, 0u, 0u};
    if (p.y)
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        const uint16_t* src = p.y + (int64_t)max(t[i], 0) * p.ldy + c;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int n = p.C - c - 32 * b;
          if (!EDGE || n >= 8) y[i][b] = load16(src + 32 * b);
          else y[i][b] = load_some(src + 32 * b, n, c + 32 * b);
        }
      }
#pragma unroll
    for (int k = 0; k < KF; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) w[k][j] = u32x4_t{0u, 0u, 0u, 0u};
    if (none) return;
    if (WT) {
      // 2 KF pieces of eight ranks x 64 columns: rank lane / 8, columns 8 (lane % 8)
#pragma unroll
      for (int k = 0; k < 2 * KF; ++k) {
        const int r = 8 * k + (lane_id() >> 3), cw = c0 + 8 * (lane_id() & 7), n = r < p.R ? p.C - cw : 0;
        const uint16_t* src = p.w + ((int64_t)group * p.R + r) * p.C + cw;
        if (EDGE ? n >= 8 : r < p.R) w[k >> 2][k & 3] = load16(src);
        else if (EDGE && n > 0) w[k >> 2][k & 3] = load_some(src, n, cw);
      }
    } else {
      const bool whole = p.R % 8 == 0;
#pragma unroll
      for (int k = 0; k < KF; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int cw = min(c0 + 32 * (j >> 1) + 8 * (i16 >> 2) + 4 * (j & 1) + (i16 & 3), p.C - 1), r = 16 * k + 8 * (q & 1);
          const uint16_t* src = p.w + ((int64_t)group * p.C + cw) * p.R + r;
          if (whole) w[k][j] = r < p.R ? load16(src) : w[k][j];
          else w[k][j] = r + 8 <= p.R ? load16(src) : load_some(src, p.R - r, cw > 8 ? 8 : cw * p.R + r);
        }
    }
  }

  // WT: from the loaded pieces to operands, through `tile` [16 KF][WT_ROW], which is this wave's alone
  DEVINL void transpose(uint16_t* tile) {
    const int i16 = lane_id() & 15, q = lane_id() >> 4;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < 2 * KF; ++k) *(u32x4_t*)(tile + (8 * k + (lane_id() >> 3)) * WT_ROW + 8 * (lane_id() & 7)) = w[k >> 2][k & 3];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < KF; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[k][j] = read_transposed(tile + (16 * k + 8 * (q & 1) + (i16 >> 2)) * WT_ROW + 32 * (j >> 1) + 8 * (i16 & 3) + 4 * (j & 1), 4 * WT_ROW * 2);
  }

  template <class H> DEVINL void finish(const ExpandParams& p, bool none, const int (&t)[MF], int c0, const H& hs, const float* row_up) {
    if (c0 + 64 <= p.C) finish<false>(p, none, t, c0, hs, row_up);
    else finish<true>(p, none, t, c0, hs, row_up);
  }
  template <bool EDGE, class H> DEVINL void finish(const ExpandParams& p, bool none, const int (&t)[MF], int c0, const H& hs, const float* row_up) {
    const int i16 = lane_id() & 15, q = lane_id() >> 4, c = c0 + 8 * q;
    wave_whole();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      f32x4_t acc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KF; ++k) {
        const u32x4_t hv = *(const u32x4_t*)&hs.pair[k][16 * i + i16][8 * q];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = mfma_16x16x32<F16>(w[k][j], hv, acc[j]);
        if (!F16) {
          u32x4_t tv = *(const u32x4_t*)&hs.third[F16 ? 0 : k][F16 ? 0 : 16 * i + i16][8 * (q & 1)];
          if (q >= 2) tv = u32x4_t{0u, 0u, 0u, 0u};
          wave_whole();
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = mfma_16x16x32<F16>(w[k][j], tv, acc[j]);
        }
      }
      const float up = row_up[16 * i + i16];
      if (t[i] >= 0) {
        uint16_t* dst = p.out + (int64_t)t[i] * p.ldo + c;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          u32x4_t o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // columns 32 b + 8 q + 2 e and the next one: fragment 2 b + e / 2, results 2 (e % 2) and the next one
            const float v0 = f32_of_16<F16>((uint16_t)(y[i][b][e] & 0xFFFFu)), v1 = f32_of_16<F16>((uint16_t)(y[i][b][e] >> 16));
            const f32x4_t& a = acc[2 * b + (e >> 1)];
            o[e] = none ? y[i][b][e] : pack_16x2<F16>(v0 + up * a[2 * (e & 1)], v1 + up * a[2 * (e & 1) + 1]);
          }
          const int n = p.C - c - 32 * b;
          if (!EDGE || n >= 8) {
            store16(dst + 32 * b, o);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < n) dst[32 * b + e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
          }
        }
      }
      wave_whole();
    }
  }
};

// v[0] + v[step] + ... of `parts` vectors `next` elements apart, in that order; MANY loads are under way at a time.
template <int MANY> DEVINL f32x4_t sum_parts(const float* part, int parts, int step, int64_t next) {
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < parts; c += MANY * step) {
    f32x4_t a[MANY];
#pragma unroll
    for (int i = 0; i < MANY; ++i) a[i] = *(const f32x4_t*)(part + min(c + i * step, parts - 1) * next);
#pragma unroll
    for (int i = 0; i < MANY; ++i)
      if (c + i * step < parts) v += a[i];
  }
  return v;
}

// h of the workgroup's rows into LDS, from `parts` sums at `part` (rows of Rp, `next` elements from part to part): four ranks
// of a row per thread; the KF * 4 threads of a row are neighbours in a wave.
template <bool F16, int KF, int MF, int THREADS, class H>
DEVINL void put_h(const ExpandParams& p, const Slot& s, bool none, bool write_h, const float* part, int parts, int64_t next, int Rp, H& hs, float* row_up) {
  const float scale = none ? 0.f : p.scales ? p.scales[s.group] : 1.f;
  for (int n = threadIdx.x; n < 16 * MF * KF * 4; n += THREADS) {
    const int row = n / (KF * 4), r = (n % (KF * 4)) * 4;
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (!none && row < s.rows && r < Rp) v = sum_parts<(MF == 1 ? 8 : 2)>(part + row * Rp + r, parts, 1, next);
    if (write_h && row < s.rows) {
      const int t = p.rows.perm[s.first + row];
      if (t >= 0 && t < p.rows.T)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r + e < p.R) p.h[(int64_t)t * p.R + r + e] = v[e];
    }
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
    uint16_t part[4][PARTS<F16>];
#pragma unroll
    for (int e = 0; e < 4; ++e) split16<F16>(v[e] * f, part[e]);
    auto put = [&](uint16_t* d, int i) {
      *(u32x2_t*)d = u32x2_t{(uint32_t)part[0][i] | ((uint32_t)part[1][i] << 16), (uint32_t)part[2][i] | ((uint32_t)part[3][i] << 16)};
    };
    put(&hs.pair[r >> 4][row][r & 15], 0);
    put(&hs.pair[r >> 4][row][16 + (r & 15)], 1);
    if (!F16) put(&hs.third[F16 ? 0 : r >> 4][F16 ? 0 : row][r & 15], PARTS<F16> - 1);
  }
}

// Rank 16: four waves to a SIMD, for which the compiler has to be asked (with three of them 73 us; transposed, where it would spill
// two registers, it makes no difference).
template <bool F16, int KF, int MF, bool WT>
__global__ __launch_bounds__(256, KF == 1 && !WT ? 4 : 1) void lora_expand(ExpandParams p, int slots) {
  __shared__ __align__(16) Parts<F16, KF, MF> hs;
  __shared__ float row_up[16 * MF];
  __shared__ __align__(16) uint16_t tiles[WT ? 4 : 1][WT ? 16 * KF : 1][WT_ROW];
  const int block = blockIdx.x / slots;
  const Slot s = find_slot(p.rows, blockIdx.x - block * slots, 16 * MF);
  if (s.group < 0) return;
  const bool none = s.group == p.rows.G - 1;
  const int64_t c_begin = (int64_t)block * p.cols;
  const int c_end = (int)min((int64_t)p.C, c_begin + p.cols);
  int c0 = (int)c_begin + 64 * wave_id();
  int t[MF];
  lane_rows<MF>(p.rows, s, t);
  Strip<F16, KF, MF, WT> strip;
  if (c0 < c_end) strip.load(p, s.group, none, t, c0);  // under way while h is put together
  put_h<F16, KF, MF, 256>(p, s, none, p.h && block == 0, p.part + (int64_t)s.padded * p.Rp, p.splits, (int64_t)p.P * p.Rp, p.Rp, hs, row_up);
  __syncthreads();
  if (none && p.out == p.y) return;
  for (; c0 < c_end; c0 += 256) {
    if (c0 >= c_begin + 256) strip.load(p, s.group, none, t, c0);
    if (WT) strip.transpose(&tiles[WT ? wave_id() : 0][0][0]);
    strip.finish(p, none, t, c0, hs, row_up);
  }
}

// ---- shrink and expand in one, for a few rows ---------------------------------------------------------------------------
// Every workgroup of 16 rows and `cols` columns computes its rows' h again: that costs K R / 16 waves of loads from L2, which
// is less than a second launch and a round trip through memory as long as A is small (see one_kernel).
template <bool F16, int NF>
__global__ __launch_bounds__(1024) void lora_few(ShrinkParams f, ExpandParams p, int slots) {
  __shared__ __align__(16) Parts<F16, NF, 1> hs;
  __shared__ float row_up[16];
  __shared__ __align__(16) float parts[16][16][16 * NF];
  const int block = blockIdx.x / slots;
  const Slot s = find_slot(p.rows, blockIdx.x - block * slots, 16);
  if (s.group < 0) return;
  const int lane = lane_id(), wave = wave_id(), i16 = lane & 15, q = lane >> 4;
  const bool none = s.group == p.rows.G - 1;
  const int c0 = block * p.cols + 64 * wave;
  const bool mine = 64 * wave < p.cols && c0 < p.C;
  int t[1];
  lane_rows<1>(p.rows, s, t);
  Strip<F16, NF, 1, false> strip;
  if (mine) strip.load(p, s.group, none, t, c0);
  if (!none) {
    const uint16_t* xr[1];
    const uint16_t* wr[NF];
    shrink_rows<1>(p.rows, s, f.x, f.ldx, xr);
    shrink_weights<NF>(s, f.w, f.ldw, f.R, wr);
    f32x4_t acc[1][NF];
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[0][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int64_t begin = (int64_t)wave * f.per_wave;
    shrink_columns<F16, NF, 1, (NF == 1 ? 4 : 2)>(xr, wr, (int)min(begin, (int64_t)f.C), (int)min((int64_t)f.C, begin + f.per_wave), q, acc);
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 4 * q + e, r = 16 * j + i16;
        parts[wave][n][r] = n < s.rows && r < f.R ? acc[0][j][e] : 0.f;
      }
  }
  __syncthreads();
  put_h<F16, NF, 1, 1024>(p, s, none, p.h && block == 0, &parts[0][0][0], 16, 16 * 16 * NF, 16 * NF, hs, row_up);
  __syncthreads();
  if (mine && !(none && p.out == p.y)) strip.finish(p, none, t, c0, hs, row_up);
}

// ---- backward: the sum of many parts ------------------------------------------------------------------------------------
// out[row][r] = the parts' sum. A workgroup takes 32 rows, a thread four ranks of one of them; the parts are dealt to as many
// strands of threads as there are threads for, whose sums meet in LDS.
__global__ __launch_bounds__(1024) void lora_sum(const float* parts, int splits, Rows rows, int Rp, int P, float* out) {
  __shared__ f32x4_t strands[1024];
  const Slot s = find_slot(rows, blockIdx.x, 32);
  if (s.group < 0 || s.group == rows.G - 1) return;
  const int n = threadIdx.x & 31, quads = Rp / 4, quad = (threadIdx.x >> 5) % quads, strand = (threadIdx.x >> 5) / quads;
  const int many = 32 / quads;  // Rp <= 128: at least one strand
  const int64_t next = (int64_t)P * Rp, at = (int64_t)(s.padded + n) * Rp + 4 * quad;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  if (strand < many && n < s.rows) v = sum_parts<8>(parts + at + strand * next, splits - strand, many, next);
  strands[threadIdx.x] = v;
  __syncthreads();
  if (strand > 0 || n >= s.rows) return;
  for (int i = 1; i < many; ++i) v += strands[threadIdx.x + 32 * quads * i];
  *(f32x4_t*)(out + at) = v;
}

// ---- backward: wgrad ----------------------------------------------------------------------------------------------------
// grad[c, r] = sum over the rows of an adapter of big[row, c] * s_g small[row, r]. A workgroup takes up to `chunk` rows, 256
// columns (64 to a wave) and up to 64 ranks, in steps of 32 rows: the rows go through LDS as they are and are read back
// transposed; the small operand is split into its parts on the way into LDS, where it lies as the matrix instruction wants it.
// fp16: four ranks of a step share a power of two that suits their largest value; a step's products are summed apart and
// scaled back. An adapter of one chunk is finished here, one without rows is cleared; the sums of several chunks are added in
// their order by lora_grad_sum.
// OUT: big is the output's gradient, small h, grad is gB as [C, R], and the same rows give the columns' share of u = gout B,
// part u[block]: wave w multiplies rows 16 (w % 2) .. of a step with columns 128 (w / 2) .., whose B it keeps in registers
// as operands, and the two halves of the columns meet in LDS one step later. Not OUT: big is x, small u, grad is gA as [R, C].
// Bound by the steps' barriers and latency: OUT on 4096 x 14336 bf16, rank 16, 44 us (3.2 TB/s with what it writes of u), x of 4096 x 4096
// 14 us. Ranks 32, 64 and 128 take 64, 128 and 216 us for OUT: u's shares grow with the rank, from 64 on one wave to a SIMD is left, and
// beyond 64 the rows are read once more. Loads two steps ahead (49 us, registers), steps of 64 rows (46 us) and chunks of 256 rows (42 us) were no faster.
struct GradParams {
  const uint16_t* big;
  int64_t ld;
  const float* small;  // by_row: [T, pitch] in row order, else `parts` of [P, pitch]
  int pitch, parts, by_row;
  const float* scales;
  uint16_t* grad;      // [L, C, R] or [L, R, C]
  float* part;         // [entries][C * R]
  const uint16_t* b;   // OUT: [L, C, R]
  float* u;            // OUT: [blocks][P][Rp]
  Rows rows;
  int C, R, Rp, P, chunk, slots, blocks;
};

constexpr int GRAD_ROW = 272;   // elements from row to row in LDS (256 columns and 32 bytes to spread the banks)
constexpr int GRAD_SKEW = 64;   // and after every eight rows
DEVINL int grad_off(int row) { return row * GRAD_ROW + (row >> 3) * GRAD_SKEW; }
constexpr int GRAD_TILE = 32 * GRAD_ROW + 4 * GRAD_SKEW;

template <bool F16, int RF, bool OUT>
__global__ __launch_bounds__(256) void lora_grad(GradParams p) {
  constexpr int SL = (RF * 128 + 255) / 256;  // four ranks of one of 32 rows: RF * 128 of them in a step
  __shared__ __align__(16) uint16_t tile[2][GRAD_TILE];
  __shared__ __align__(16) uint16_t small[2][PARTS<F16>][RF * 16][32];
  __shared__ float small_up[2][RF * 4];
  __shared__ f32x4_t half_u[OUT ? 2 : 1][OUT ? 2 * RF : 1][64];
  const int slot = blockIdx.x % p.slots, block = blockIdx.x / p.slots % p.blocks, r0 = blockIdx.x / p.slots / p.blocks * 16 * RF;
  const Slot s = find_slot(p.rows, slot, p.chunk, false);
  const int tid = threadIdx.x, lane = lane_id(), wave = wave_id(), i16 = lane & 15, q = lane >> 4;
  const int c0 = block * 256, rows16 = (s.rows + 15) & ~15;
  const int64_t block_size = (int64_t)p.C * p.R;
  if (s.of == p.rows.G - 1) return;
  uint16_t* grad = p.grad + s.of * block_size;
  if (s.group < 0) {
    if (s.size <= 0 && r0 == 0) {  // the one slot of an adapter without rows
      const int cols = min(256, p.C - c0), row = OUT ? cols * p.R : cols, pieces = (row + 7) / 8;  // its share: rows of so many elements
      uint16_t* first = grad + (OUT ? (int64_t)c0 * p.R : (int64_t)c0);
      for (int n = tid; n < pieces * (OUT ? 1 : p.R); n += 256) {
        const int r = n / pieces, at = 8 * (n - r * pieces);
        uint16_t* d = first + (int64_t)r * p.C + at;
        if (at + 8 <= row) store16(d, u32x4_t{0u, 0u, 0u, 0u});
        else
          for (int e = 0; e < row - at; ++e) d[e] = 0;
      }
    }
    return;
  }
  const int cl = c0 + 8 * (tid & 31), some = p.C - cl;  // this thread's eight columns of the rows tid / 32 + 8 j
  const float scale = p.scales ? p.scales[s.group] : 1.f;

  f32x4_t acc[4][RF], au[RF];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int f = 0; f < RF; ++f) acc[j][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // rows of the step at n: t[0..3] of the big operand, t[4] of the small one (row tid % 32)
  auto row_of = [&](int n, int (&t)[5]) {
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const int m = n + (j < 4 ? (tid >> 5) + 8 * j : (tid & 31));
      t[j] = m < s.rows ? p.rows.perm[s.first + m] : -1;
      if (t[j] >= p.rows.T) t[j] = -1;
    }
  };
  u32x4_t bv[4];
  f32x4_t sv[SL];
  const bool edge = c0 + 256 > p.C;
  auto load = [&](int n0, const int (&t)[5]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bv[j] = u32x4_t{0u, 0u, 0u, 0u};
      const uint16_t* src = p.big + (int64_t)max(t[j], 0) * p.ld + cl;
      if (!edge) bv[j] = t[j] >= 0 ? load16(src) : bv[j];
      else if (t[j] >= 0) bv[j] = some >= 8 ? load16(src) : load_some(src, some, cl);
    }
#pragma unroll
    for (int j = 0; j < SL; ++j) {
      const int i = tid + 256 * j, n = n0 + (i & 31), r = r0 + 4 * (i >> 5);
      sv[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (i >= RF * 128 || t[4] < 0 || r >= p.R) continue;
      const float* src = p.small + (int64_t)(p.by_row ? t[4] : s.padded + n) * p.pitch + r;
      if (r + 4 > p.pitch) {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (r + e < p.pitch) sv[j][e] = src[e];
      } else {
        sv[j] = *(const f32x4_any_t*)src;
        if (p.parts > 1) sv[j] = sum_parts<8>(src, p.parts, 1, (int64_t)p.P * p.pitch);
      }
    }
  };
  auto put_small = [&](int buf) {
#pragma unroll
    for (int j = 0; j < SL; ++j) {
      const int i = tid + 256 * j, n = i & 31, r = 4 * (i >> 5);
      if (i >= RF * 128) continue;
      f32x4_t v = sv[j];
      float f = 1.f;
      if (F16) {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = finite_max(m, v[e] * scale);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) m = max(m, __shfl_xor(m, d, 64));
        f = pow2_down(m);
        if (n == 0) small_up[buf][r >> 2] = pow2_up(m);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t part[PARTS<F16>];
        split16<F16>(v[e] * scale * f, part);
#pragma unroll
        for (int h = 0; h < PARTS<F16>; ++h) small[buf][h][r + e][n] = part[h];
      }
    }
  };
  // this wave's share of u for the rows of the step before, waves 0 and 1: with the other half's
  auto write_u = [&](int n0) {
    const int n = n0 + 16 * wave;
    if (wave < 2 && n < rows16) {
      float* u = p.u + ((int64_t)block * p.P + s.padded + n) * p.Rp + r0;
#pragma unroll
      for (int f = 0; f < RF; ++f) {
        const f32x4_t v = au[f] + half_u[(n0 >> 5) & 1][wave * RF + f][lane];
        if (r0 + 16 * f < p.Rp)
#pragma unroll
          for (int e = 0; e < 4; ++e) u[(int64_t)(4 * q + e) * p.Rp + 16 * f + i16] = v[e];
      }
    }
  };
  int t[5];
  row_of(0, t);
  // B of this wave's 128 columns, ranks r0 ..: through the tile, one half of the columns after the other. Its loads and the
  // first step's are under way together.
  u32x4_t bt[OUT ? 4 : 1][RF], staged[OUT ? 2 : 1][RF];
  constexpr int ROW = RF * 16 + 8;
  static_assert(128 * ROW <= 2 * GRAD_TILE, "128 columns of B fit the tiles");
  if (OUT)
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < RF; ++i) {
        const int n = tid + 256 * i, c = c0 + 128 * half + n / (RF * 2), r = r0 + 8 * (n % (RF * 2));
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (c < p.C) {
          const uint16_t* src = p.b + ((int64_t)s.group * p.C + c) * p.R + r;
          if (r + 8 <= p.R) v = load16(src);
          else if (r < p.R) v = load_some(src, p.R - r, c > 8 ? 8 : c * p.R + r);
        }
        staged[OUT ? half : 0][i] = v;
      }
  load(0, t);
  row_of(32, t);
  if (OUT) {
    uint16_t* at = tile[0];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < RF; ++i) {
        const int n = tid + 256 * i;
        *(u32x4_t*)(at + (n / (RF * 2)) * ROW + 8 * (n % (RF * 2))) = staged[OUT ? half : 0][i];
      }
      __syncthreads();
      if ((wave >> 1) == half)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int f = 0; f < RF; ++f) bt[OUT ? k : 0][f] = read_transposed(at + (32 * k + 8 * q + (i16 >> 2)) * ROW + 16 * f + 4 * (i16 & 3), 4 * ROW * 2);
      __syncthreads();
    }
  }
  int buf = 0;
  for (int n0 = 0; n0 < s.rows; n0 += 32, buf ^= 1) {
    uint16_t* tl = tile[buf];
#pragma unroll
    for (int j = 0; j < 4; ++j) *(u32x4_t*)(tl + grad_off((tid >> 5) + 8 * j) + 8 * (tid & 31)) = bv[j];
    wave_whole();
    put_small(buf);
    __syncthreads();
    // stores before loads: a wave waits for its memory operations in their order, and the next step waits for these loads
    if (OUT && n0 > 0) write_u(n0 - 32);
    if (n0 + 32 < s.rows) {
      load(n0 + 32, t);
      row_of(n0 + 64, t);
    }
    if (OUT) {
#pragma unroll
      for (int f = 0; f < RF; ++f) au[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32x4_t v = *(const u32x4_t*)(tl + grad_off(16 * (wave & 1) + i16) + 128 * (wave >> 1) + 32 * k + 8 * q);
#pragma unroll
        for (int f = 0; f < RF; ++f) au[f] = mfma_16x16x32<F16>(v, bt[OUT ? k : 0][f], au[f]);
      }
      if (wave >= 2)
#pragma unroll
        for (int f = 0; f < RF; ++f) half_u[(n0 >> 5) & 1][(wave - 2) * RF + f][lane] = au[f];
    }
    u32x4_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      b[j] = read_transposed(tl + grad_off(8 * q + (i16 >> 2)) + 64 * wave + 16 * j + 4 * (i16 & 3), 4 * GRAD_ROW * 2);
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      u32x4_t v[PARTS<F16>];
#pragma unroll
      for (int h = 0; h < PARTS<F16>; ++h) v[h] = *(const u32x4_t*)&small[buf][h][16 * f + i16][8 * q];
      if (F16) {
        const float up = small_up[buf][4 * f + (OUT ? q : i16 >> 2)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < PARTS<F16>; ++h) d = OUT ? mfma_16x16x32<F16>(v[h], b[j], d) : mfma_16x16x32<F16>(b[j], v[h], d);
          acc[j][f] += d * up;
        }
      } else {
#pragma unroll
        for (int h = 0; h < PARTS<F16>; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j][f] = OUT ? mfma_16x16x32<F16>(v[h], b[j], acc[j][f]) : mfma_16x16x32<F16>(b[j], v[h], acc[j][f]);
      }
    }
  }
  if (OUT) {
    __syncthreads();
    write_u((s.rows - 1) & ~31);
  }
  const bool whole = s.size <= p.chunk;
  const int64_t entry = s.begin / (p.chunk / 2) + (s.first - s.begin) / p.chunk;
  float* part = p.part + entry * block_size;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      const int c = c0 + 64 * wave + 16 * j + (OUT ? i16 : 4 * q), r = r0 + 16 * f + (OUT ? 4 * q : i16);
      if (c >= p.C || r >= p.R) continue;
      const f32x4_t v = acc[j][f];
      const int64_t at = OUT ? (int64_t)c * p.R + r : (int64_t)r * p.C + c;
      const int n = min(4, OUT ? p.R - r : p.C - c);
      if (n == 4) {
        if (whole) *(u32x2_any_t*)(grad + at) = u32x2_t{pack_16x2<F16>(v[0], v[1]), pack_16x2<F16>(v[2], v[3])};
        else *(f32x4_any_t*)(part + at) = v;
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

// The gradients of adapters of several chunks, of both products; a thread takes eight elements.
template <bool F16>
__global__ __launch_bounds__(256) void lora_grad_sum(GradParams p0, GradParams p1, int blocks0) {
  const int g = blockIdx.y;
  const bool first = (int)blockIdx.x < blocks0;
  const Rows rows = p0.rows;
  const int chunk = first ? p0.chunk : p1.chunk, C = first ? p0.C : p1.C;
  const int begin = clamp_off(rows, g), size = clamp_off(rows, g + 1) - begin;
  if (size <= chunk) return;
  const int64_t block_size = (int64_t)C * p0.R;
  const int64_t i = ((int64_t)(blockIdx.x - (first ? 0 : blocks0)) * 256 + threadIdx.x) * 8;
  if (i >= block_size) return;
  const int n = (int)min((int64_t)8, block_size - i);
  const int chunks = (size + chunk - 1) / chunk;
  const float* part = (first ? p0.part : p1.part) + (int64_t)(begin / (chunk / 2)) * block_size + i;
  uint16_t* d = (first ? p0.grad : p1.grad) + g * block_size + i;
  if (n == 8) {
    f32x4_t v[2] = {};
    for (int c = 0; c < chunks; c += 4) {  // four chunks' loads under way together
      f32x4_t a[4][2];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int b = 0; b < 2; ++b) a[k][b] = *(const f32x4_any_t*)(part + min(c + k, chunks - 1) * block_size + 4 * b);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < chunks) v[0] += a[k][0], v[1] += a[k][1];
    }
    store16(d, u32x4_t{pack_16x2<F16>(v[0][0], v[0][1]), pack_16x2<F16>(v[0][2], v[0][3]), pack_16x2<F16>(v[1][0], v[1][1]), pack_16x2<F16>(v[1][2], v[1][3])});
    return;
  }
  for (int e = 0; e < n; ++e) {
    float v = 0.f;
    for (int c = 0; c < chunks; ++c) v += part[c * block_size + e];
    d[e] = cvt_16<F16>(v);
  }
}

int slots_of(int64_t T, int64_t G, int unit) { return (int)(T == 0 ? 1 : T < T / unit + G ? T : T / unit + G); }

template <bool F16, int NF, int MF>
void launch_shrink(const ShrinkParams& p, hipStream_t stream) {
  const int slots = slots_of(p.rows.T, p.rows.G, 16 * MF);
  hipLaunchKernelGGL((lora_shrink<F16, NF, MF>), dim3(slots * p.splits), dim3(512), 0, stream, p, slots);
}

template <bool F16, int KF, int MF, bool WT>
void launch_expand(const ExpandParams& p, hipStream_t stream) {
  const int slots = slots_of(p.rows.T, p.rows.G, 16 * MF);
  hipLaunchKernelGGL((lora_expand<F16, KF, MF, WT>), dim3(slots * ((p.C + p.cols - 1) / p.cols)), dim3(256), 0, stream, p, slots);
}

int rank_blocks(int R) { return R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8; }
int64_t tiles_of(int64_t T, int64_t G, int rows) { return T / rows + (G < T ? G : T); }
// Rows per workgroup of shrink and expand: 64 (32 for the highest ranks) use an adapter's weights for more rows, 16 give more
// workgroups. 64 once those, with 256 of the C columns each, fill the card.
int rows_of(int64_t T, int R, int C) {
  const int many = rank_blocks(R) == 8 ? 32 : 64;
  return T / many * ((C + 255) / 256) >= 256 ? many : 16;
}

template <bool F16>
void shrink(const ShrinkParams& p, hipStream_t stream) {
  const bool many = rows_of(p.rows.T, p.R, p.C) > 16;
  switch (rank_blocks(p.R)) {
    case 1: many ? launch_shrink<F16, 1, 4>(p, stream) : launch_shrink<F16, 1, 1>(p, stream); break;
    case 2: many ? launch_shrink<F16, 2, 4>(p, stream) : launch_shrink<F16, 2, 1>(p, stream); break;
    case 4: many ? launch_shrink<F16, 4, 4>(p, stream) : launch_shrink<F16, 4, 1>(p, stream); break;
    default: many ? launch_shrink<F16, 8, 2>(p, stream) : launch_shrink<F16, 8, 1>(p, stream); break;
  }
}

// Columns per workgroup of expand: 1024 (four strips per wave) once that fills the card, else 256.
template <bool F16, bool WT>
void expand(ExpandParams p, hipStream_t stream) {
  const int rows = rows_of(p.rows.T, p.R, p.C);
  const bool many = rows > 16;
  p.cols = tiles_of(p.rows.T, p.rows.G, rows) * ((p.C + 1023) / 1024) >= 512 ? 1024 : 256;
  switch (rank_blocks(p.R)) {
    case 1: many ? launch_expand<F16, 1, 4, WT>(p, stream) : launch_expand<F16, 1, 1, WT>(p, stream); break;
    case 2: many ? launch_expand<F16, 2, 4, WT>(p, stream) : launch_expand<F16, 2, 1, WT>(p, stream); break;
    case 4: many ? launch_expand<F16, 4, 4, WT>(p, stream) : launch_expand<F16, 4, 1, WT>(p, stream); break;
    default: many ? launch_expand<F16, 8, 2, WT>(p, stream) : launch_expand<F16, 8, 1, WT>(p, stream); break;
  }
}

// Columns per wave of shrink, a multiple of 64: the reduced axis is split until there are about 1024 workgroups, into at most
// 16 parts, which the next kernel adds again for every row.
int shrink_per_wave(int64_t T, int64_t G, int R, int C) {
  int64_t s = 1024 / (tiles_of(T, G, rows_of(T, R, C)) + 1);
  s = s < 1 ? 1 : s > 16 ? 16 : s;
  return (int)((C + 512 * s - 1) / (512 * s) * 64);
}
int splits_of(int C, int per_wave) { return (C + 8 * per_wave - 1) / (8 * per_wave); }

// Columns per workgroup of the one kernel: 256 (four of its waves), doubled while there are more than two workgroups to a CU.
int one_kernel_cols(int64_t T, int64_t G, int N) {
  int cols = 256;
  while (cols < 1024 && tiles_of(T, G, 16) * ((N + cols - 1) / cols) > 512) cols *= 2;
  return cols;
}
// One kernel while sixteen waves read a workgroup's share of A and x in one go (256 columns each) and all workgroups together read
// at most 64 MB from L2. 4 rows of 4096 -> 14336, rank 16: 9 us against 3.8 + 5.5 us and a second launch, which costs the host
// 5 us; 277 rows of 6336 -> 320: 20 us against 17, 64 rows of 14336 -> 4096: 23 us against 8 + 6 us.
bool one_kernel(int64_t T, int64_t G, int K, int N, int R) {
  if (T > 512 || R > 32 || K > 4096) return false;
  const int cols = one_kernel_cols(T, G, N);
  return tiles_of(T, G, 16) * ((N + cols - 1) / cols) * K * (32 * (1 + rank_blocks(R))) <= 64 << 20;
}

// Rows of a workgroup of wgrad: 512, or half or a quarter of that until there are about 400 workgroups, but 512 where that is all
// there is, which saves the kernel that adds the chunks. Beyond 8192 rows also twice, four times .. as many while more than 768
// workgroups are left, since every chunk of an adapter of several costs a set of partial sums. One adapter, rank 16, all of the
// backward pass: 65536 rows of 256 columns 150 us with 128 rows to a workgroup and 411 with 4096 (32 workgroups); 16384 of 4096 171
// with 512 and 207 with 1024; 8192 of 4096 -> 14336, 16 adapters of rank 64, 418 with 512 and 424 with 1024.
int grad_chunk(int64_t T, int C) {
  if (T <= 512) return 512;
  const int64_t blocks = (C + 255) / 256;
  int chunk = 512;
  while (chunk > 128 && T / chunk * blocks < 384) chunk /= 2;
  while (T > 8192 && chunk >= 512 && T / (2 * chunk) * blocks >= 768) chunk *= 2;
  return chunk;
}
int64_t grad_entries(int64_t T, int chunk) { return T / (chunk / 2); }

struct Sizes {
  int64_t G, P, Rp, blocks;
  int chunk[2];  // rows of a workgroup of wgrad on the output's gradient and on x
  int s_x, w_x;  // shrink of x: splits, columns per wave
};
Sizes sizes_of(int64_t T, int L, int K, int N, int R) {
  Sizes z;
  z.G = L + 1;
  z.P = 16 * (T / 16 + z.G);
  z.Rp = (R + 15) / 16 * 16;
  z.blocks = (N + 255) / 256;
  z.chunk[0] = grad_chunk(T, N);
  z.chunk[1] = grad_chunk(T, K);
  z.w_x = shrink_per_wave(T, z.G, R, K);
  z.s_x = splits_of(K, z.w_x);
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

// With few column blocks the readers of u add its parts themselves.
bool sum_first(const Sizes& z) { return z.blocks > 8; }

struct BackwardSpace {
  float *part_u, *part_h, *sum_u, *sums[2];
};
BackwardSpace backward_space(Workspace& w, const Sizes& z, int64_t T, int K, int N, int R, bool with_h) {
  BackwardSpace b;
  b.part_u = w.take<float>(z.blocks * z.P * z.Rp);
  b.part_h = with_h ? nullptr : w.take<float>(z.s_x * z.P * z.Rp);
  b.sum_u = sum_first(z) ? w.take<float>(z.P * z.Rp) : b.part_u;
  b.sums[0] = w.take<float>(grad_entries(T, z.chunk[0]) * N * R);
  b.sums[1] = w.take<float>(grad_entries(T, z.chunk[1]) * K * R);
  return b;
}

// ids outside [0, L) become L, the group of rows without an adapter.
__global__ __launch_bounds__(256) void lora_keys(const int32_t* ids, int32_t* keys, int T, int L) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < T) keys[t] = ids[t] >= 0 && ids[t] < L ? ids[t] : L;
}

ShrinkParams shrink_params(const LoraParams& p, const Rows& rows, const Sizes& z, float* part) {
  ShrinkParams f{};
  f.x = (const uint16_t*)p.x; f.ldx = p.ldx; f.w = (const uint16_t*)p.a; f.ldw = p.K; f.part = part; f.rows = rows;
  f.C = p.K; f.R = p.R; f.Rp = (int)z.Rp; f.P = (int)z.P; f.per_wave = z.w_x; f.splits = z.s_x;
  return f;
}

template <bool F16>
void forward(const LoraParams& p, hipStream_t stream) {
  const Sizes z = sizes_of(p.T, p.L, p.K, p.N, p.R);
  const Rows rows{p.perm, p.offsets, (int)z.G, p.T};
  ShrinkParams f = shrink_params(p, rows, z, (float*)p.workspace);
  ExpandParams e{};
  e.part = f.part; e.w = (const uint16_t*)p.b; e.scales = p.scales; e.y = (const uint16_t*)p.y; e.ldy = p.ldy; e.out = (uint16_t*)p.out;
  e.ldo = p.ldo; e.h = (float*)p.h; e.rows = rows; e.C = p.N; e.R = p.R; e.Rp = (int)z.Rp; e.P = (int)z.P; e.splits = z.s_x;
  if (one_kernel(p.T, z.G, p.K, p.N, p.R)) {
    const int slots = slots_of(p.T, z.G, 16);
    f.per_wave = (p.K + 1023) / 1024 * 64;
    e.cols = one_kernel_cols(p.T, z.G, p.N);
    const dim3 grid(slots * ((p.N + e.cols - 1) / e.cols)), block(1024);
    if (p.R <= 16) hipLaunchKernelGGL((lora_few<F16, 1>), grid, block, 0, stream, f, e, slots);
    else hipLaunchKernelGGL((lora_few<F16, 2>), grid, block, 0, stream, f, e, slots);
    return;
  }
  if (p.L > 0) shrink<F16>(f, stream);
  expand<F16, false>(e, stream);
}

template <bool F16, bool OUT>
void launch_grad(const GradParams& g, hipStream_t stream) {
  const int rf = rank_blocks(g.R) > 4 ? 4 : rank_blocks(g.R);
  const dim3 grid(g.slots * g.blocks * ((g.R + 16 * rf - 1) / (16 * rf))), block(256);
  if (rf == 1) hipLaunchKernelGGL((lora_grad<F16, 1, OUT>), grid, block, 0, stream, g);
  else if (rf == 2) hipLaunchKernelGGL((lora_grad<F16, 2, OUT>), grid, block, 0, stream, g);
  else hipLaunchKernelGGL((lora_grad<F16, 4, OUT>), grid, block, 0, stream, g);
}

template <bool F16>
void backward(const LoraParams& p, hipStream_t stream) {
  const Sizes z = sizes_of(p.T, p.L, p.K, p.N, p.R);
  Workspace w{(char*)p.workspace, 0};
  const BackwardSpace b = backward_space(w, z, p.T, p.K, p.N, p.R, p.h != nullptr);
  const Rows rows{p.perm, p.offsets, (int)z.G, p.T};
  ExpandParams e{};
  e.part = b.sum_u; e.w = (const uint16_t*)p.a; e.scales = p.scales; e.y = (const uint16_t*)p.gx_in; e.ldy = p.gx_in ? p.ld_gx_in : p.ld_gx;
  e.out = (uint16_t*)p.gx; e.ldo = p.ld_gx; e.rows = rows; e.C = p.K; e.R = p.R; e.Rp = (int)z.Rp; e.P = (int)z.P; e.splits = 1;
  if (p.L == 0) return expand<F16, true>(e, stream);
  if (!p.h) shrink<F16>(shrink_params(p, rows, z, b.part_h), stream);
  e.splits = sum_first(z) ? 1 : (int)z.blocks;
  GradParams g[2] = {};
  for (int j = 0; j < 2; ++j) {  // 0: gB and u from the output's gradient and h; 1: gA from x and u
    g[j].big = (const uint16_t*)(j ? p.x : p.y); g[j].ld = j ? p.ldx : p.ldy;
    g[j].small = j ? b.sum_u : p.h ? (const float*)p.h : b.part_h;
    g[j].by_row = !j && p.h; g[j].pitch = g[j].by_row ? p.R : (int)z.Rp; g[j].parts = j ? e.splits : p.h ? 1 : z.s_x;
    g[j].scales = p.scales; g[j].grad = (uint16_t*)(j ? p.grad_a : p.grad_b); g[j].part = b.sums[j]; g[j].b = (const uint16_t*)p.b; g[j].u = b.part_u;
    g[j].rows = rows; g[j].C = j ? p.K : p.N; g[j].R = p.R; g[j].Rp = (int)z.Rp; g[j].P = (int)z.P;
    g[j].chunk = z.chunk[j]; g[j].slots = (int)(p.T / z.chunk[j] + z.G); g[j].blocks = (g[j].C + 255) / 256;
  }
  launch_grad<F16, true>(g[0], stream);
  if (sum_first(z))
    hipLaunchKernelGGL(lora_sum, dim3(slots_of(p.T, z.G, 32)), dim3(1024), 0, stream, (const float*)b.part_u, (int)z.blocks, rows, (int)z.Rp, (int)z.P, b.sum_u);
  launch_grad<F16, false>(g[1], stream);
  expand<F16, true>(e, stream);
  if (p.T > z.chunk[0] || p.T > z.chunk[1]) {  // adapters of several chunks are possible
    const int blocks0 = (int)(((int64_t)p.N * p.R + 2047) / 2048), blocks1 = (int)(((int64_t)p.K * p.R + 2047) / 2048);
    hipLaunchKernelGGL((lora_grad_sum<F16>), dim3(blocks0 + blocks1, p.L), dim3(256), 0, stream, g[0], g[1], blocks0);
  }
}

}  // namespace

size_t lora_forward_workspace(int64_t T, int L, int K, int N, int R) {
  if (one_kernel(T, L + 1, K, N, R)) return 0;
  const Sizes z = sizes_of(T, L, K, N, R);
  return (size_t)z.s_x * z.P * z.Rp * sizeof(float);
}

size_t lora_backward_workspace(int64_t T, int L, int K, int N, int R, bool with_h) {
  Workspace w{nullptr, 0};
  backward_space(w, sizes_of(T, L, K, N, R), T, K, N, R, with_h);
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
