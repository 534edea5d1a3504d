// Gated delta rule: a recurrence whose state is a K x V matrix per head and which overwrites what it holds under a key.
// Per sequence b, head h and step t, time-major:
//
//   q^ = q / sqrt(|q|^2 + eps),  k^ = k / sqrt(|k|^2 + eps)     (eps = 1e-6)
//   al = exp(A softplus(a + dt_bias)),  be = sigmoid(b)
//   S_t = al S_{t-1} + k^ (be (v - (al S_{t-1})^T k^))^T
//   y_t = scale S_t^T q^
//
// A step after the end of an episode starts from a cleared state. H / Hk heads share the rows of q and k.
//
// Sequences go in chunks of CH steps (32 for bf16, 16 for fp32). With G_i the sum of log al up to step i of the chunk and
// D_ij = exp(G_i - G_j), 0 where an episode starts in j+1..i (D_i0: from the chunk's start, D_cj: to its end), the
// written values U solve a unit lower triangular system, and the rest is products:
//
//   (I + M) U = Y = be (V - D_i0 K S_0),   M_ij = be_i D_ij k^_i k^_j (j < i)
//   O = scale D_i0 Q S_0 + P U,            P_ij = scale D_ij q^_i k^_j (j <= i)
//   S_c = D_c0 S_0 + K^T (D_cj U)
//
// T = (I + M)^-1 is formed by substitution in diagonal blocks of 16 (its elements stay below one, since every step
// contracts; powers of M do not), the blocks below by products. The gradient, from dS_c and dO, in reverse order:
//
//   dU = P^T dO + D_cj K dS_c,  dY = T^T dU,  dV = be dY,  db = <dY, U> (1 - be)
//   E_ij = scale D_ij dO_i U_j (j <= i),  F_ij = -be_i D_ij dY_i U_j (j < i)
//   dQ^ = scale D_i0 dO S_0^T + E K^
//   dK^ = (-D_i0 be dY S_0^T + F K^) + (F^T K^ + E^T Q^ + D_cj U dS_c^T)      (as row i, as row j of M and P)
//   dlog al_t = sum_{j < t <= i} (P_ij dO_i U_j - M_ij dY_i U_j) + sum_{i >= t} (what of <q^, dQ^> + <k^, dK^> comes from S_0)
//             + sum_{j < t} (what of <k^, dK^> comes from dS_c) + D_c0 <S_0, dS_c>: every pair whose decay t is a factor of
//   dS_0 = D_c0 dS_c + Q^T (scale D_i0 dO) - K^T (D_i0 be dY)
//
// Steps hidden by an episode's start are selected away: D is 0 there and what it multiplies is dropped, so an infinite
// state does not pass. Inside the products 0 times a non-finite U would; a chunk that holds an episode's start and finds a
// non-finite value is done again episode by episode, with the other rows zero.
//
// Layout. A block owns one head of one sequence, wavefront w the state's columns 16 w .. 16 w + 15 (gradient: rows of the
// transposed state too), in the accumulator layout of the 16x16 matrix instructions: lane l holds rows 4 (l / 16) + r, column
// l % 16. That layout is also the one of the instruction's right operand when the contraction runs over
// those rows, so S, U and dY go from one product to the next without leaving the registers, and all of a wavefront's chain
// stays in its columns. bf16 rows enter the products as they are (their norms are factors outside) and values
// held in fp32 as the sum of two bf16, 16 bits of them; fp32 takes the fp32 matrix instructions.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "routes.hpp"

#include <type_traits>

namespace ph {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

constexpr float kEps = 1e-6f;
constexpr double kLog2e = 1.4426950408889634;

struct Args {
  long T, B, units;  // units: sequences x heads
  int Hk, H, K, V;
  const void *q, *k, *v, *a, *b;
  long q_t, q_b, q_h, k_t, k_b, k_h, v_t, v_b, v_h, a_t, a_b, b_t, b_b;
  const float *A, *dt_bias, *done, *first, *h0;
  float scale;
  int vec;  // rows of q, k, v (and dy) can be read 16 bytes at a time
  void* y;
  long y_t, y_b, y_h;
  float *h_out, *keep;
};

struct GradArgs {
  const void* dy;
  long dy_t, dy_b, dy_h;
  const float *keep, *dh;
  void *dq, *dk, *dv, *da, *db;
  long dq_t, dq_b, dq_h, dk_t, dk_b, dk_h, dv_t, dv_b, dv_h, da_t, da_b, db_t, db_b;
  float* dh0;
  float *qpart, *kpart;  // [T][B][H][K] of every value head, where heads share their keys
  float* gpart;          // [2][H][B]: sums of dlog al softplus and of dlog al A sigmoid
};

// ---- elements ------------------------------------------------------------------------------------------
__device__ __forceinline__ float ldf(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ void stf(uint16_t* p, float v) { *p = bf16_rne(v); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ float ex2(float v) { return __builtin_amdgcn_exp2f(v); }
// softplus, max(v, 0) + log(1 + e) with e = exp(-|v|). What rounding 1 + e to w dropped is added back as it is, so small e
// keep their digits.
__device__ __forceinline__ float softplus(float v) {
  const float e = ex2(-fabsf(v) * (float)kLog2e), w = 1.f + e;
  return fmaxf(v, 0.f) + fmaf(__builtin_amdgcn_logf(w), (float)(1 / kLog2e), e - (w - 1.f));
}
__device__ __forceinline__ float sigma(float v) { return 1.f / (1.f + ex2(v * -(float)kLog2e)); }
// max and comparisons with a NaN drop it; a gate of NaN stays one
__device__ __forceinline__ float log_decay(float A, float sp) {
  const float g = A * sp;
  return g < -1e9f ? -1e9f : g;  // differences of sums stay numbers
}
__device__ __forceinline__ bool finite(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7f800000u) != 0x7f800000u; }

// ---- matrix operands -------------------------------------------------------------------------------------
// Operands are taken in units of 16 of the contraction, of which lane l holds 4 (l / 16) + 0..3.
template <bool BF> struct Elem { using type = uint16_t; using unit = s4; static constexpr int CH = 32, pad = 8, V = 8; };
template <> struct Elem<false> { using type = float; using unit = f4; static constexpr int CH = 16, pad = 4, V = 4; };

// acc += a b over N units. bf16 units go in pairs where there are two.
template <int N> __device__ __forceinline__ f4 dot(const s4* a, const s4* b, f4 acc) {
#pragma unroll
  for (int i = 0; i + 1 < N; i += 2) {
    const s8 x = __builtin_shufflevector(a[i], a[i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    const s8 y = __builtin_shufflevector(b[i], b[i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), acc, 0, 0, 0);
  }
  if constexpr (N & 1) acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a[N - 1], b[N - 1], acc, 0, 0, 0);
  return acc;
}
template <int N> __device__ __forceinline__ f4 dot(const f4* a, const f4* b, f4 acc) {
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][r], b[i][r], acc, 0, 0, 0);
  return acc;
}

// fp32 values as operands: for bf16 the nearest bf16 and what it leaves, also rounded to bf16 (the sum is within 2^-17 of
// the value), else the values themselves.
template <bool BF> struct Pair {
  s4 hi, lo;
  __device__ __forceinline__ void set(f4 v) {
    const uint32_t a = bf16x2_rne(v[0], v[1]), b = bf16x2_rne(v[2], v[3]);
    hi = __builtin_bit_cast(s4, u2{a, b});
    const float h0 = __builtin_bit_cast(float, a << 16), h1 = __builtin_bit_cast(float, a & 0xffff0000u);
    const float h2 = __builtin_bit_cast(float, b << 16), h3 = __builtin_bit_cast(float, b & 0xffff0000u);
    lo = __builtin_bit_cast(s4, u2{bf16x2_rne(v[0] - h0, v[1] - h1), bf16x2_rne(v[2] - h2, v[3] - h3)});
  }
};
template <> struct Pair<false> {
  f4 hi;
  __device__ __forceinline__ void set(f4 v) { hi = v; }
};
// acc += a b: a exact rows and b of pairs, and both of pairs (the product of the two remainders is below what they keep).
template <bool BF, int N>
__device__ __forceinline__ f4 dot2(const typename Elem<BF>::unit* a, const Pair<BF>* b, f4 acc) {
  typename Elem<BF>::unit h[N];
#pragma unroll
  for (int i = 0; i < N; i++) h[i] = b[i].hi;
  acc = dot<N>(a, h, acc);
  if constexpr (BF) {
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = b[i].lo;
    acc = dot<N>(a, h, acc);
  }
  return acc;
}
template <bool BF, int N> __device__ __forceinline__ f4 dot3(const Pair<BF>* a, const Pair<BF>* b, f4 acc) {
  typename Elem<BF>::unit h[N];
  if constexpr (BF) {
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = a[i].lo;
    typename Elem<BF>::unit g[N];
#pragma unroll
    for (int i = 0; i < N; i++) g[i] = b[i].hi;
    acc = dot<N>(h, g, acc);
  }
#pragma unroll
  for (int i = 0; i < N; i++) h[i] = a[i].hi;
  return dot2<BF, N>(h, b, acc);
}
// acc += a b: a of pairs, b exact columns.
template <bool BF, int N>
__device__ __forceinline__ f4 dot2r(const Pair<BF>* a, const typename Elem<BF>::unit* b, f4 acc) {
  typename Elem<BF>::unit h[N];
#pragma unroll
  for (int i = 0; i < N; i++) h[i] = a[i].hi;
  acc = dot<N>(h, b, acc);
  if constexpr (BF) {
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = a[i].lo;
    acc = dot<N>(h, b, acc);
  }
  return acc;
}

// Units of a matrix in LDS, leading dimension LD. row_unit: row `row` + l % 16, columns `col` + 4 (l / 16) + 0..3 (left
// operand with the contraction over columns, or the right one of the transposed matrix); col_unit: rows `row` + 4 (l / 16) +
// 0..3, column `col` + l % 16 (contraction over rows), for 16-bit elements by the transposing load, which gives lane l of
// sixteen the column l of the four rows that the sixteen lanes' addresses cover.
template <int LD> __device__ __forceinline__ s4 row_unit(const uint16_t* m, int row, int col) {
  const int l = threadIdx.x & 63;
  return *reinterpret_cast<const s4*>(m + (row + (l & 15)) * LD + col + 4 * (l >> 4));
}
template <int LD> __device__ __forceinline__ f4 row_unit(const float* m, int row, int col) {
  const int l = threadIdx.x & 63;
  return *reinterpret_cast<const f4*>(m + (row + (l & 15)) * LD + col + 4 * (l >> 4));
}
template <int LD> __device__ __forceinline__ s4 col_unit(const uint16_t* m, int row, int col) {
  const int l = threadIdx.x & 63;
  const uint16_t* p = m + (row + 4 * (l >> 4) + ((l & 15) >> 2)) * LD + col + 4 * (l & 3);
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
}
template <int LD> __device__ __forceinline__ f4 col_unit(const float* m, int row, int col) {
  const int l = threadIdx.x & 63;
  const float* p = m + (row + 4 * (l >> 4)) * LD + col + (l & 15);
  return f4{p[0], p[LD], p[2 * LD], p[3 * LD]};
}
__device__ __forceinline__ f4 widen(s4 v) {
  return f4{bf16_to_f32((uint16_t)v[0]), bf16_to_f32((uint16_t)v[1]), bf16_to_f32((uint16_t)v[2]), bf16_to_f32((uint16_t)v[3])};
}
__device__ __forceinline__ f4 widen(f4 v) { return v; }

// ---- a chunk's rows ------------------------------------------------------------------------------------
// The 16 bytes of a row of W columns that a thread stages: row tid / (P / V), columns from V (tid % (P / V)) on; zero where
// the row or the columns end.
template <bool BF, int P, typename T = typename Elem<BF>::type>
__device__ __forceinline__ u4 load_row(const T* base, long stride, int rows, int W, bool vec) {
  constexpr int V = Elem<BF>::V;
  const int row = threadIdx.x / (P / V), c = threadIdx.x % (P / V) * V;
  u4 r = {0, 0, 0, 0};
  if (row < rows && c < W) {
    const T* p = base + row * stride + c;
    if (vec) {
      r = *reinterpret_cast<const u4*>(p);
    } else {
      T v[V];
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = c + i < W ? p[i] : T(0);
      __builtin_memcpy(&r, v, 16);
    }
  }
  return r;
}
template <bool BF> __device__ __forceinline__ float square_sum(u4 r) {
  float s = 0.f;
  if constexpr (BF) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float x = __builtin_bit_cast(float, r[i] << 16), y = __builtin_bit_cast(float, r[i] & 0xffff0000u);
      s = fmaf(x, x, fmaf(y, y, s));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t u = r[i];
      const float x = __builtin_bit_cast(float, u);
      s = fmaf(x, x, s);
    }
  }
  return s;
}
template <bool BF> __device__ __forceinline__ bool all_finite(u4 r) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t u = r[i];
    if constexpr (BF) ok = ok && (u & 0x7f80u) != 0x7f80u && (u & 0x7f800000u) != 0x7f800000u;
    else ok = ok && (u & 0x7f800000u) != 0x7f800000u;
  }
  return ok;
}

// What the chunk's rows have in common, by row.
template <int CH> struct Rows {
  double G[CH];                       // base-2 logarithm of the decay from the chunk's start
  int seg[CH];                        // starts of episodes up to the row
  float be[CH], rq[CH], rk[CH];       // write strength, 1 / norms
  float d0[CH], dc[CH];               // D_i0, D_cj
  float sp[CH], arg[CH];              // softplus and its argument (gradient)
  float c0, pad;                      // D_c0
  int starts;                         // bit i: row i starts an episode
};

// The lane's row of the gates, loaded ahead.
struct Gate {
  float a, b, start;
};
template <typename T> __device__ __forceinline__ Gate load_gate(const Args& s, long bt, int h, long t0, int rows, int i) {
  Gate g = {0.f, 0.f, 0.f};
  if (i < rows) {
    const long t = t0 + i;
    g.a = ldf((const T*)s.a + t * s.a_t + bt * s.a_b + h) + (s.dt_bias ? s.dt_bias[h] : 0.f);
    g.b = ldf((const T*)s.b + t * s.b_t + bt * s.b_b + h);
    if (t > 0) g.start = s.done ? s.done[(t - 1) * s.B + bt] : 0.f;
    else g.start = s.first ? s.first[bt] : 0.f;
  }
  return g;
}
// Fills r for rows lo..hi-1 from the gates of wavefront 0's lanes (all of it calls).
template <int CH> __device__ __forceinline__ void fill_rows(Rows<CH>& r, const Gate& g, float A, int lo, int hi) {
  const int i = threadIdx.x;
  const bool in = i >= lo && i < hi;
  const float sp = softplus(g.a);
  double G = in ? (double)log_decay(A, sp) * kLog2e : 0.0;
  const unsigned long long starts = __ballot(in && g.start != 0.f);
#pragma unroll
  for (int d = 1; d < CH; d *= 2) {
    const double o = __shfl_up(G, d);
    if (i >= d) G += o;
  }
  const double last = __shfl(G, CH - 1);
  if (i < CH) {
    const int seg = __popcll(starts & ((2ull << i) - 1)), all = __popcll(starts);
    r.G[i] = G;
    r.seg[i] = seg;
    r.be[i] = in ? sigma(g.b) : 0.f;
    r.sp[i] = sp;
    r.arg[i] = g.a;
    const float d0 = ex2((float)G), dc = ex2((float)(last - G));
    r.d0[i] = in && seg == 0 ? d0 : 0.f;
    r.dc[i] = in && seg == all ? dc : 0.f;
    if (i == CH - 1) {
      r.c0 = all == 0 ? d0 : 0.f;
      r.starts = (int)(starts & 0xffffffffu);
    }
  }
}
__device__ __forceinline__ f4 rows4(const float* r, int at) { return *reinterpret_cast<const f4*>(r + at + 4 * ((threadIdx.x & 63) >> 4)); }
// c x where c is not zero: what a start hides may be anything
__device__ __forceinline__ f4 sel_mul(f4 c, f4 x) {
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = c[i] == 0.f ? 0.f : c[i] * x[i];
  return x;
}

// M (and P, transposed by the reader) of the chunk: tiles on and below the diagonal, dealt out over the wavefronts.
template <bool BF, int P, int LD>
__device__ __forceinline__ void score_tiles(const Rows<Elem<BF>::CH>& r, const typename Elem<BF>::type* Qs,
                                            const typename Elem<BF>::type* Ks, float* Mm, float* Pm, float scale) {
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, NT = P / 16, CP = CH + 4, TILES = NB * (NB + 1) / 2;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int id = w; id < 2 * TILES; id += NT) {
    const bool isP = id >= TILES;
    const int tile = isP ? id - TILES : id, bi = tile == 0 ? 0 : 1, bj = tile == 2 ? 1 : 0;  // (0,0) (1,0) (1,1)
    typename Elem<BF>::unit x[NT], y[NT];
#pragma unroll
    for (int m = 0; m < NT; m++) {
      x[m] = row_unit<LD>(isP ? Qs : Ks, 16 * bi, 16 * m);
      y[m] = row_unit<LD>(Ks, 16 * bj, 16 * m);
    }
    f4 acc = dot<NT>(x, y, f4{0.f, 0.f, 0.f, 0.f});
    const int j = 16 * bj + (l & 15);
    const double Gj = r.G[j];
    const int segj = r.seg[j];
    const float rkj = r.rk[j];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int i = 16 * bi + 4 * (l >> 4) + k;
      const bool on = segj == r.seg[i] && (isP ? j <= i : j < i);
      const float c = ex2((float)(r.G[i] - Gj)) * rkj * (isP ? scale * r.rq[i] : r.be[i] * r.rk[i]);
      (isP ? Pm : Mm)[i * CP + j] = on ? c * acc[k] : 0.f;
    }
  }
}

// The diagonal blocks of (I + M)^-1 into Tm, one column per lane of wavefront 0.
template <int CH> __device__ __forceinline__ void invert_blocks(const float* Mm, float* Tm) {
  constexpr int CP = CH + 4;
  const int l = threadIdx.x;
  if (l >= CH) return;
  const int o = l & ~15, c = l & 15;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    float s = i == c ? 1.f : 0.f;
#pragma unroll
    for (int j4 = 0; j4 < i; j4 += 4) {
      const f4 m = *reinterpret_cast<const f4*>(Mm + (o + i) * CP + o + j4);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (j4 + k < i) s = fmaf(-m[k], x[j4 + k], s);
    }
    x[i] = s;
    Tm[(o + i) * CP + o + c] = s;
  }
}

// U = T Y by blocks, T's blocks below the diagonal through M.
template <bool BF> __device__ __forceinline__ void solve(const float* Tm, const float* Mm, const f4* Y, f4* U) {
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, CP = CH + 4;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  Pair<BF> t, y, u;
  t.set(row_unit<CP>(Tm, 0, 0));
  y.set(Y[0]);
  U[0] = dot3<BF, 1>(&t, &y, zero);
  if constexpr (NB == 2) {
    u.set(-U[0]);
    t.set(row_unit<CP>(Mm, 16, 0));
    y.set(dot3<BF, 1>(&t, &u, Y[1]));
    t.set(row_unit<CP>(Tm, 16, 16));
    U[1] = dot3<BF, 1>(&t, &y, zero);
  }
}
// dY = T^T dU
template <bool BF> __device__ __forceinline__ void solve_t(const float* Tm, const float* Mm, const f4* dU, f4* dY) {
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, CP = CH + 4;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  Pair<BF> t, y;
  f4 top = dU[0];
  if constexpr (NB == 2) {
    y.set(dU[1]);
    t.set(col_unit<CP>(Tm, 16, 16));
    dY[1] = dot3<BF, 1>(&t, &y, zero);
    y.set(-dY[1]);
    t.set(col_unit<CP>(Mm, 16, 0));
    top = dot3<BF, 1>(&t, &y, top);
  }
  y.set(top);
  t.set(col_unit<CP>(Tm, 0, 0));
  dY[0] = dot3<BF, 1>(&t, &y, zero);
}

// Tile m of a [K][V] matrix's column block w: rows 16 m + 4 (l / 16) + 0..3, column 16 w + l % 16; zero outside.
__device__ __forceinline__ f4 state_tile(const float* s, int K, int V, int m, int w) {
  const int l = threadIdx.x & 63, r = 16 * m + 4 * (l >> 4), c = 16 * w + (l & 15);
  f4 x = {0.f, 0.f, 0.f, 0.f};
  if (s && c < V) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (r + i < K) x[i] = s[(long)(r + i) * V + c];
  }
  return x;
}
__device__ __forceinline__ void put_state_tile(float* s, int K, int V, int m, int w, f4 x) {
  const int l = threadIdx.x & 63, r = 16 * m + 4 * (l >> 4), c = 16 * w + (l & 15);
  if (c < V) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (r + i < K) s[(long)(r + i) * V + c] = x[i];
  }
}
// The transposed matrix's tile m of block w: columns of V 16 m + 4 (l / 16) + 0..3, row 16 w + l % 16.
__device__ __forceinline__ f4 state_tile_t(const float* s, int K, int V, int m, int w) {
  const int l = threadIdx.x & 63, c = 16 * m + 4 * (l >> 4), r = 16 * w + (l & 15);
  f4 x = {0.f, 0.f, 0.f, 0.f};
  if (s && r < K) {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (c + i < V) x[i] = s[(long)r * V + c + i];
  }
  return x;
}

template <bool BF, int P, typename T = typename Elem<BF>::type>
__device__ __forceinline__ void put_row(T* tile, u4 r, int lo, int hi) {
  constexpr int V = Elem<BF>::V, LD = P + Elem<BF>::pad;
  const int row = threadIdx.x / (P / V), c = threadIdx.x % (P / V) * V;
  if (row < lo || row >= hi) r = u4{0, 0, 0, 0};
  *reinterpret_cast<u4*>(tile + row * LD + c) = r;
}
// 1 / sqrt(|row|^2 + eps) of the staged rows, 0 for those left out
template <bool BF, int P> __device__ __forceinline__ void put_norm(float* out, u4 r, int lo, int hi) {
  constexpr int L = P / Elem<BF>::V;  // lanes of a row
  float s = square_sum<BF>(r);
#pragma unroll
  for (int d = 1; d < L; d *= 2) s += __shfl_xor(s, d);
  const int row = threadIdx.x / L;
  if (threadIdx.x % L == 0) out[row] = row >= lo && row < hi ? 1.f / sqrtf(s + kEps) : 0.f;
}

// ---- sequences ------------------------------------------------------------------------------------------
template <bool BF, int P> __global__ void __launch_bounds__(4 * P) k_delta_fwd(const Args s) {
  using T = typename Elem<BF>::type;
  using unit = typename Elem<BF>::unit;
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, NT = P / 16, LD = P + Elem<BF>::pad, CP = CH + 4;
  __shared__ __attribute__((aligned(16))) T Qs[CH * LD], Ks[CH * LD], Vs[CH * LD];
  __shared__ __attribute__((aligned(16))) float Mm[CH * CP], Tm[CH * CP], Pm[CH * CP];
  __shared__ Rows<CH> R;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  for (long unit_id = blockIdx.x; unit_id < s.units; unit_id += gridDim.x) {
    const long bt = unit_id / s.H;
    const int h = (int)(unit_id % s.H), hk = h / (s.H / s.Hk);
    const T* qp = (const T*)s.q + bt * s.q_b + hk * s.q_h;
    const T* kp = (const T*)s.k + bt * s.k_b + hk * s.k_h;
    const T* vp = (const T*)s.v + bt * s.v_b + h * s.v_h;
    T* yp = (T*)s.y + bt * s.y_b + h * s.y_h;
    const long kv = (long)s.K * s.V;
    const float A = s.A[h];
    f4 S[NT];
#pragma unroll
    for (int m = 0; m < NT; m++) S[m] = state_tile(s.h0 ? s.h0 + unit_id * kv : nullptr, s.K, s.V, m, w);
    for (long t0 = 0; t0 < s.T; t0 += CH) {
      const int rows = (int)(s.T - t0 < CH ? s.T - t0 : CH);
      if (s.keep) {
#pragma unroll
        for (int m = 0; m < NT; m++) put_state_tile(s.keep + (t0 / CH * s.units + unit_id) * kv, s.K, s.V, m, w, S[m]);
      }
      const u4 q = load_row<BF, P>(qp + t0 * s.q_t, s.q_t, rows, s.K, s.vec);
      const u4 k = load_row<BF, P>(kp + t0 * s.k_t, s.k_t, rows, s.K, s.vec);
      const u4 v = load_row<BF, P>(vp + t0 * s.v_t, s.v_t, rows, s.V, s.vec);
      Gate g;
      if (w == 0) g = load_gate<T>(s, bt, h, t0, rows, l);
      for (int lo = 0, hi = rows; lo < rows;) {
        __syncthreads();  // the rows before have been read
        put_row<BF, P>(Qs, q, lo, hi);
        put_row<BF, P>(Ks, k, lo, hi);
        put_row<BF, P>(Vs, v, lo, hi);
        put_norm<BF, P>(R.rq, q, lo, hi);
        put_norm<BF, P>(R.rk, k, lo, hi);
        __syncthreads();
        if (w == 0) fill_rows<CH>(R, g, A, lo, hi);
        __syncthreads();
        score_tiles<BF, P, LD>(R, Qs, Ks, Mm, Pm, s.scale);
        __syncthreads();
        if (w == 0) invert_blocks<CH>(Mm, Tm);
        Pair<BF> Sp[NT];
#pragma unroll
        for (int m = 0; m < NT; m++) Sp[m].set(S[m]);
        f4 Y[NB], O[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) {
          unit x[NT];
#pragma unroll
          for (int m = 0; m < NT; m++) x[m] = row_unit<LD>(Ks, 16 * n, 16 * m);
          const f4 ks = dot2<BF, NT>(x, Sp, zero);
          Y[n] = rows4(R.be, 16 * n) * (widen(col_unit<LD>(Vs, 16 * n, 16 * w)) - sel_mul(rows4(R.d0, 16 * n) * rows4(R.rk, 16 * n), ks));
#pragma unroll
          for (int m = 0; m < NT; m++) x[m] = row_unit<LD>(Qs, 16 * n, 16 * m);
          O[n] = sel_mul(s.scale * rows4(R.d0, 16 * n) * rows4(R.rq, 16 * n), dot2<BF, NT>(x, Sp, zero));
        }
        __syncthreads();
        f4 U[NB];
        solve<BF>(Tm, Mm, Y, U);
        const int inside = R.starts & ~(1 << lo);
        if (inside) {
          bool bad = false;
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) bad |= !finite(U[n][i]);
          if (__syncthreads_or(bad)) {
            hi = __ffs(inside) - 1;
            continue;
          }
        }
        Pair<BF> Up[NB], x[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) Up[n].set(U[n]);
        x[0].set(row_unit<CP>(Pm, 0, 0));
        O[0] = dot3<BF, 1>(x, Up, O[0]);
        if constexpr (NB == 2) {
          x[0].set(row_unit<CP>(Pm, 16, 0));
          x[1].set(row_unit<CP>(Pm, 16, 16));
          O[1] = dot3<BF, 2>(x, Up, O[1]);
        }
        const int c = 16 * w + (l & 15);
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int row = 16 * n + 4 * (l >> 4) + i;
            if (row >= lo && row < hi && c < s.V) stf(yp + (t0 + row) * s.y_t + c, O[n][i]);
          }
#pragma unroll
        for (int n = 0; n < NB; n++) Up[n].set(sel_mul(rows4(R.dc, 16 * n) * rows4(R.rk, 16 * n), U[n]));
        const float c0 = R.c0;
#pragma unroll
        for (int m = 0; m < NT; m++) {
          unit kt[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) kt[n] = col_unit<LD>(Ks, 16 * n, 16 * m);
          S[m] = dot2<BF, NB>(kt, Up, sel_mul(f4{c0, c0, c0, c0}, S[m]));
        }
        lo = hi;
        hi = rows;
      }
    }
    if (s.h_out) {
#pragma unroll
      for (int m = 0; m < NT; m++) put_state_tile(s.h_out + unit_id * kv, s.K, s.V, m, w, S[m]);
    }
  }
}

// The gradient of one sequence's head, chunks in reverse. Wavefront w holds dS's columns 16 w .. and, for the products
// that contract over V, the transposed dS's (rows 16 w .. of dS).
template <bool BF, int P> struct BwdLds {
  using T = typename Elem<BF>::type;
  static constexpr int CH = Elem<BF>::CH, LD = P + Elem<BF>::pad, UD = CH + 4, CP = CH + 4, NT = P / 16;
  T Q[CH * LD], K[CH * LD], dO[CH * LD];
  // values of fp32 transposed, [V][step]: U and dY, for bf16 both halves. V rests where U comes: it is read before.
  union {
    T V[CH * LD];
    T U[P * UD];
    float sums[4][NT][CH];  // when U has been read: <q^, dQ^>, <k^, dK^>, the parts of S_0 and of dS_c
  };
  T dY[P * UD], Ulo[BF ? P * UD : 1], dYlo[BF ? P * UD : 1];
  union {
    float M[CH * CP];
    float F[CH * CP];
  };
  union {
    float Pm[CH * CP];
    float E[CH * CP];
  };
  union {
    float Tm[CH * CP];
    float W[CH * CP];  // P_ij dO_i U_j - M_ij dY_i U_j
  };
  float ysum[NT][CH], pairs[CH / 16][CH], tot[NT];
  Rows<CH> R;
};

// A tile's values into a transposed buffer pair at rows 16 w + l % 16, columns `at` + 4 (l / 16) + 0..3; and units of it.
template <bool BF, int UD, typename T> __device__ __forceinline__ void put_t(T* hi, T* lo, int w, int at, f4 v) {
  const int l = threadIdx.x & 63, o = (16 * w + (l & 15)) * UD + at + 4 * (l >> 4);
  Pair<BF> p;
  p.set(v);
  *reinterpret_cast<typename Elem<BF>::unit*>(hi + o) = p.hi;
  if constexpr (BF) *reinterpret_cast<s4*>(lo + o) = p.lo;
}
template <bool BF, int UD, typename T> __device__ __forceinline__ Pair<BF> col_pair(const T* hi, const T* lo, int row, int col) {
  Pair<BF> p;
  p.hi = col_unit<UD>(hi, row, col);
  if constexpr (BF) p.lo = col_unit<UD>(lo, row, col);
  return p;
}
template <bool BF, int UD, typename T> __device__ __forceinline__ Pair<BF> row_pair(const T* hi, const T* lo, int row, int col) {
  Pair<BF> p;
  p.hi = row_unit<UD>(hi, row, col);
  if constexpr (BF) p.lo = row_unit<UD>(lo, row, col);
  return p;
}
__device__ __forceinline__ float row16_sum(float v) {
  v += dpp_mov<0xB1>(v);
  v += dpp_mov<0x4E>(v);
  v += dpp_mov<0x141>(v);
  v += dpp_mov<0x140>(v);
  return v;
}

template <bool BF, int P> __global__ void __launch_bounds__(4 * P) k_delta_bwd(const Args s, const GradArgs o) {
  using T = typename Elem<BF>::type;
  using unit = typename Elem<BF>::unit;
  using Lds = BwdLds<BF, P>;
  constexpr int CH = Lds::CH, NB = CH / 16, NT = Lds::NT, LD = Lds::LD, CP = Lds::CP, UD = Lds::UD;
  constexpr int TILES = NB * (NB + 1) / 2;
  static_assert(sizeof(Lds) <= kMaxLdsBytes, "LDS of a block");
  __shared__ __attribute__((aligned(16))) Lds L;
  Rows<CH>& R = L.R;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  for (long unit_id = blockIdx.x; unit_id < s.units; unit_id += gridDim.x) {
    const long bt = unit_id / s.H;
    const int h = (int)(unit_id % s.H), hk = h / (s.H / s.Hk);
    const T* qp = (const T*)s.q + bt * s.q_b + hk * s.q_h;
    const T* kp = (const T*)s.k + bt * s.k_b + hk * s.k_h;
    const T* vp = (const T*)s.v + bt * s.v_b + h * s.v_h;
    const T* op = (const T*)o.dy + bt * o.dy_b + h * o.dy_h;
    const long kv = (long)s.K * s.V;
    const float A = s.A[h];
    double sumA = 0.0, sumB = 0.0;  // of wavefront 0's lanes
    f4 dS[NT], dSt[NT];
#pragma unroll
    for (int m = 0; m < NT; m++) {
      dS[m] = state_tile(o.dh ? o.dh + unit_id * kv : nullptr, s.K, s.V, m, w);
      dSt[m] = state_tile_t(o.dh ? o.dh + unit_id * kv : nullptr, s.K, s.V, m, w);
    }
    for (long c = (s.T + CH - 1) / CH - 1; c >= 0; c--) {
      const long t0 = c * CH;
      const int rows = (int)(s.T - t0 < CH ? s.T - t0 : CH);
      const float* S0 = o.keep + (c * s.units + unit_id) * kv;
      const u4 q = load_row<BF, P>(qp + t0 * s.q_t, s.q_t, rows, s.K, s.vec);
      const u4 k = load_row<BF, P>(kp + t0 * s.k_t, s.k_t, rows, s.K, s.vec);
      const u4 v = load_row<BF, P>(vp + t0 * s.v_t, s.v_t, rows, s.V, s.vec);
      const u4 d = load_row<BF, P>(op + t0 * o.dy_t, o.dy_t, rows, s.V, s.vec);
      Gate g;
      if (w == 0) g = load_gate<T>(s, bt, h, t0, rows, l);
      for (int lo = 0, hi = rows; hi > 0;) {
        __syncthreads();  // the rows before have been read
        put_row<BF, P>(L.Q, q, lo, hi);
        put_row<BF, P>(L.K, k, lo, hi);
        put_row<BF, P>(L.V, v, lo, hi);
        put_row<BF, P>(L.dO, d, lo, hi);
        put_norm<BF, P>(R.rq, q, lo, hi);
        put_norm<BF, P>(R.rk, k, lo, hi);
        __syncthreads();
        if (w == 0) fill_rows<CH>(R, g, A, lo, hi);
        __syncthreads();
        score_tiles<BF, P, LD>(R, L.Q, L.K, L.M, L.Pm, s.scale);
        __syncthreads();
        if (w == 0) invert_blocks<CH>(L.M, L.Tm);
        f4 Y[NB], dU[NB], sd = zero;
        {
          Pair<BF> Sp[NT], Dp[NT];
#pragma unroll
          for (int m = 0; m < NT; m++) {
            const f4 S = state_tile(S0, s.K, s.V, m, w);
            sd += S * dS[m];
            Sp[m].set(S);
            Dp[m].set(dS[m]);
          }
#pragma unroll
          for (int n = 0; n < NB; n++) {
            unit x[NT];
#pragma unroll
            for (int m = 0; m < NT; m++) x[m] = row_unit<LD>(L.K, 16 * n, 16 * m);
            Y[n] = rows4(R.be, 16 * n) * (widen(col_unit<LD>(L.V, 16 * n, 16 * w)) -
                                          sel_mul(rows4(R.d0, 16 * n) * rows4(R.rk, 16 * n), dot2<BF, NT>(x, Sp, zero)));
            dU[n] = sel_mul(rows4(R.dc, 16 * n) * rows4(R.rk, 16 * n), dot2<BF, NT>(x, Dp, zero));
          }
        }
        __syncthreads();
        // dU, dY, U: this wavefront's columns of V
        f4 U[NB], dY[NB];
        unit dOc[NB];
        {
          solve<BF>(L.Tm, L.M, Y, U);
          Pair<BF> x[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) dOc[n] = col_unit<LD>(L.dO, 16 * n, 16 * w);
          x[0].set(col_unit<CP>(L.Pm, 0, 0));
          if constexpr (NB == 2) {
            x[1].set(col_unit<CP>(L.Pm, 16, 0));
            dU[0] = dot2r<BF, 2>(x, dOc, dU[0]);
            x[0].set(col_unit<CP>(L.Pm, 16, 16));
            dU[1] = dot2r<BF, 1>(x, dOc + 1, dU[1]);
          } else {
            dU[0] = dot2r<BF, 1>(x, dOc, dU[0]);
          }
          solve_t<BF>(L.Tm, L.M, dU, dY);
        }
        const int inside = R.starts & ~(1 << lo);
        if (inside) {
          const int row = threadIdx.x / (P / Elem<BF>::V);
          bool bad = row >= lo && row < hi && (!all_finite<BF>(q) || !all_finite<BF>(d));
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) bad |= !finite(U[n][i]) || !finite(dY[n][i]);
          if (__syncthreads_or(bad)) {
            lo = 31 - __clz(inside);
            continue;
          }
        }
        const int col = 16 * w + (l & 15);
#pragma unroll
        for (int n = 0; n < NB; n++) {
          const f4 be = rows4(R.be, 16 * n);
          put_t<BF, UD>(L.U, L.Ulo, w, 16 * n, U[n]);
          put_t<BF, UD>(L.dY, L.dYlo, w, 16 * n, dY[n]);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int row = 16 * n + 4 * (l >> 4) + i;
            if (o.dv && row >= lo && row < hi && col < s.V)
              stf((T*)o.dv + bt * o.dv_b + h * o.dv_h + (t0 + row) * o.dv_t + col, be[i] * dY[n][i]);
            const float sum = row16_sum(dY[n][i] * U[n][i]);
            if ((l & 15) == 0) L.ysum[w][row] = sum;
          }
        }
        const float c0 = R.c0;
        float tot = c0 == 0.f ? 0.f : c0 * (sd[0] + sd[1] + sd[2] + sd[3]);
        // dS of the chunk's start; the transposed one below, when its old values have been used
        {
          Pair<BF> x[NB], y[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) {
            x[n].set(sel_mul(s.scale * rows4(R.d0, 16 * n) * rows4(R.rq, 16 * n), widen(dOc[n])));
            y[n].set(sel_mul(-rows4(R.d0, 16 * n) * rows4(R.rk, 16 * n) * rows4(R.be, 16 * n), dY[n]));
          }
#pragma unroll
          for (int m = 0; m < NT; m++) {
            unit a[NB];
#pragma unroll
            for (int n = 0; n < NB; n++) a[n] = col_unit<LD>(L.Q, 16 * n, 16 * m);
            dS[m] = dot2<BF, NB>(a, x, sel_mul(f4{c0, c0, c0, c0}, dS[m]));
#pragma unroll
            for (int n = 0; n < NB; n++) a[n] = col_unit<LD>(L.K, 16 * n, 16 * m);
            dS[m] = dot2<BF, NB>(a, y, dS[m]);
          }
        }
        __syncthreads();
        for (int tile = w; tile < TILES; tile += NT) {
          const int bi = tile == 0 ? 0 : 1, bj = tile == 2 ? 1 : 0;  // (0,0) (1,0) (1,1)
          f4 e = zero, f = zero;
          {
            Pair<BF> y[NT], x[NT];
            unit z[NT];
#pragma unroll
            for (int m = 0; m < NT; m++) {
              y[m] = col_pair<BF, UD>(L.U, L.Ulo, 16 * m, 16 * bj);
              z[m] = row_unit<LD>(L.dO, 16 * bi, 16 * m);
              x[m] = col_pair<BF, UD>(L.dY, L.dYlo, 16 * m, 16 * bi);
            }
            e = dot2<BF, NT>(z, y, e);
            f = dot3<BF, NT>(x, y, f);
          }
          const int j = 16 * bj + (l & 15);
          const double Gj = R.G[j];
          const int segj = R.seg[j];
#pragma unroll
          for (int i4 = 0; i4 < 4; i4++) {
            const int i = 16 * bi + 4 * (l >> 4) + i4, at = i * CP + j;
            const bool on = segj == R.seg[i] && j <= i;
            const float d = ex2((float)(R.G[i] - Gj));
            L.W[at] = on && j < i ? L.Pm[at] * e[i4] - L.M[at] * f[i4] : 0.f;
            L.E[at] = on ? d * s.scale * e[i4] : 0.f;
            L.F[at] = on && j < i ? -d * R.be[i] * f[i4] : 0.f;
          }
        }
        // products over V for this wavefront's columns of K: dO S_0^T, dY S_0^T, U dS^T
        f4 X1[NB], X2[NB], X3[NB];
        {
          Pair<BF> St[NT], Dt[NT];
#pragma unroll
          for (int m = 0; m < NT; m++) {
            St[m].set(state_tile_t(S0, s.K, s.V, m, w));
            Dt[m].set(dSt[m]);
          }
#pragma unroll
          for (int n = 0; n < NB; n++) {
            unit x[NT];
#pragma unroll
            for (int m = 0; m < NT; m++) x[m] = row_unit<LD>(L.dO, 16 * n, 16 * m);
            X1[n] = sel_mul(s.scale * rows4(R.d0, 16 * n), dot2<BF, NT>(x, St, zero));
            Pair<BF> y[NT];
#pragma unroll
            for (int m = 0; m < NT; m++) y[m] = col_pair<BF, UD>(L.dY, L.dYlo, 16 * m, 16 * n);
            X2[n] = sel_mul(-rows4(R.d0, 16 * n) * rows4(R.be, 16 * n), dot3<BF, NT>(y, St, zero));
#pragma unroll
            for (int m = 0; m < NT; m++) y[m] = col_pair<BF, UD>(L.U, L.Ulo, 16 * m, 16 * n);
            X3[n] = sel_mul(rows4(R.dc, 16 * n), dot3<BF, NT>(y, Dt, zero));
          }
        }
        unit Kc[NB], Qc[NB];  // this wavefront's columns of K and Q
#pragma unroll
        for (int n = 0; n < NB; n++) {
          Kc[n] = col_unit<LD>(L.K, 16 * n, 16 * w);
          Qc[n] = col_unit<LD>(L.Q, 16 * n, 16 * w);
        }
        {
          Pair<BF> x[NB], y[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) {
            x[n].set(sel_mul(s.scale * rows4(R.d0, 16 * n) * rows4(R.rq, 16 * n), widen(Qc[n])));
            y[n].set(sel_mul(-rows4(R.d0, 16 * n) * rows4(R.rk, 16 * n) * rows4(R.be, 16 * n), widen(Kc[n])));
          }
#pragma unroll
          for (int m = 0; m < NT; m++) {
            unit a[NB];
#pragma unroll
            for (int n = 0; n < NB; n++) a[n] = col_unit<LD>(L.dO, 16 * n, 16 * m);
            dSt[m] = dot2<BF, NB>(a, x, sel_mul(f4{c0, c0, c0, c0}, dSt[m]));
            Pair<BF> b[NB];
#pragma unroll
            for (int n = 0; n < NB; n++) b[n] = row_pair<BF, UD>(L.dY, L.dYlo, 16 * m, 16 * n);
            dSt[m] = dot3<BF, NB>(b, y, dSt[m]);
          }
        }
        __syncthreads();
        // E K, F K (rows as i), F^T K, E^T Q (rows as j); the norms' factors go into E and F
        f4 dQ[NB], dKi[NB], dKj[NB];
        {
          f4 rk[NB], rq[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) {
            rk[n] = rows4(R.rk, 16 * n);
            rq[n] = rows4(R.rq, 16 * n);
          }
#pragma unroll
          for (int n = 0; n < NB; n++) {
            Pair<BF> e[NB], f[NB];
#pragma unroll
            for (int m = 0; m <= n; m++) {
              e[m].set(row_unit<CP>(L.E, 16 * n, 16 * m) * rk[m]);
              f[m].set(row_unit<CP>(L.F, 16 * n, 16 * m) * rk[m]);
            }
            if (n == 0) {
              dQ[n] = dot2r<BF, 1>(e, Kc, zero);
              dKi[n] = dot2r<BF, 1>(f, Kc, zero);
            } else {
              dQ[n] = dot2r<BF, NB>(e, Kc, zero);
              dKi[n] = dot2r<BF, NB>(f, Kc, zero);
            }
#pragma unroll
            for (int m = n; m < NB; m++) {
              e[m].set(col_unit<CP>(L.E, 16 * m, 16 * n) * rq[m]);
              f[m].set(col_unit<CP>(L.F, 16 * m, 16 * n) * rk[m]);
            }
            if (n == NB - 1) {
              dKj[n] = dot2r<BF, 1>(f + n, Kc + n, dot2r<BF, 1>(e + n, Qc + n, zero));
            } else {
              dKj[n] = dot2r<BF, NB>(f, Kc, dot2r<BF, NB>(e, Qc, zero));
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NB; n++) {
          const f4 qn = widen(Qc[n]) * rows4(R.rq, 16 * n), kn = widen(Kc[n]) * rows4(R.rk, 16 * n);
          const f4 from0 = qn * X1[n] + kn * X2[n], fromc = kn * X3[n];
          dQ[n] += X1[n];
          dKi[n] += X2[n];
          dKi[n] += dKj[n] + X3[n];
          const f4 sq = qn * dQ[n], sk = kn * dKi[n];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float v[4] = {row16_sum(sq[i]), row16_sum(sk[i]), row16_sum(from0[i]), row16_sum(fromc[i])};
            if ((l & 15) == 0) {
#pragma unroll
              for (int e = 0; e < 4; e++) L.sums[e][w][16 * n + 4 * (l >> 4) + i] = v[e];
            }
          }
        }
        // sums over the pairs j < t <= i, rows t: a triangle of ones times W, then along the row
        for (int tile = w; tile < TILES; tile += NT) {
          const int bt = tile == 0 ? 0 : 1, bj = tile == 2 ? 1 : 0, t = 16 * bt + (l & 15);
          f4 acc = zero;
          for (int m = bt; m < NB; m++) {
            f4 ones;
#pragma unroll
            for (int i = 0; i < 4; i++) ones[i] = 16 * m + 4 * (l >> 4) + i >= t ? 1.f : 0.f;
            const f4 x = m == bt && bj > bt ? zero : col_unit<CP>(L.W, 16 * m, 16 * bj);
            acc = dot<1>(&ones, &x, acc);
          }
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int row = 16 * bt + 4 * (l >> 4) + i;
            const float sum = row16_sum(16 * bj + (l & 15) < row ? acc[i] : 0.f);
            if ((l & 15) == 0) L.pairs[bj][row] = sum;
          }
        }
        tot = group_sum<64>(tot);
        if (l == 0) L.tot[w] = tot;
        __syncthreads();
        // through the norms
#pragma unroll
        for (int n = 0; n < NB; n++) {
          const f4 rq = rows4(R.rq, 16 * n), rk = rows4(R.rk, 16 * n);
          f4 sq = zero, sk = zero;
#pragma unroll
          for (int m = 0; m < NT; m++) {
            sq += rows4(L.sums[0][m], 16 * n);
            sk += rows4(L.sums[1][m], 16 * n);
          }
          const f4 dq = rq * (dQ[n] - widen(Qc[n]) * rq * sq), dk = rk * (dKi[n] - widen(Kc[n]) * rk * sk);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int row = 16 * n + 4 * (l >> 4) + i;
            if (row < lo || row >= hi || col >= s.K) continue;
            if (o.qpart) {
              const long at = (((t0 + row) * s.B + bt) * s.H + h) * s.K + col;
              o.qpart[at] = dq[i];
              o.kpart[at] = dk[i];
            } else {
              if (o.dq) stf((T*)o.dq + bt * o.dq_b + h * o.dq_h + (t0 + row) * o.dq_t + col, dq[i]);
              if (o.dk) stf((T*)o.dk + bt * o.dk_b + h * o.dk_h + (t0 + row) * o.dk_t + col, dk[i]);
            }
          }
        }
        if (w == 0) {  // the gates
          float from0 = 0.f, fromc = 0.f, dbr = 0.f, all = 0.f;
          const int i = l < CH ? l : CH - 1;
#pragma unroll
          for (int m = 0; m < NT; m++) {
            from0 += L.sums[2][m][i];
            fromc += L.sums[3][m][i];
            dbr += L.ysum[m][i];
            all += L.tot[m];
          }
          if (l >= CH) from0 = fromc = 0.f;
#pragma unroll
          for (int e = 1; e < CH; e *= 2) {  // of the rows from t on, of the rows up to t
            const float x = __shfl_down(from0, e), y = __shfl_up(fromc, e);
            if (l + e < CH) from0 += x;
            if (l >= e) fromc += y;
          }
          fromc = __shfl_up(fromc, 1);
          if (l == 0) fromc = 0.f;
          float dg = L.pairs[0][i] + from0 + fromc + all;
          if (NB == 2 && i >= 16) dg += L.pairs[NB - 1][i];
          if (l >= lo && l < hi) {
            const float be = R.be[l], arg = R.arg[l];
            const float da = dg * A * sigma(arg);
            if (o.da) stf((T*)o.da + (t0 + l) * o.da_t + bt * o.da_b + h, da);
            if (o.db) stf((T*)o.db + (t0 + l) * o.db_t + bt * o.db_b + h, dbr * (1.f - be));
            sumA += (double)dg * (double)R.sp[l];
            sumB += (double)da;
          }
        }
        if (R.starts >> lo & 1) {  // nothing passes to the steps before, whatever these hold
#pragma unroll
          for (int m = 0; m < NT; m++) dS[m] = dSt[m] = zero;
        }
        hi = lo;
        lo = 0;
      }
    }
    if (o.dh0) {
#pragma unroll
      for (int m = 0; m < NT; m++) put_state_tile(o.dh0 + unit_id * kv, s.K, s.V, m, w, dS[m]);
    }
    if (w == 0 && o.gpart) {
#pragma unroll
      for (int e = 1; e < CH; e *= 2) {
        sumA += __shfl_xor(sumA, e);
        sumB += __shfl_xor(sumB, e);
      }
      if (l == 0) {
        o.gpart[(long)h * s.B + bt] = (float)sumA;
        o.gpart[((long)s.H + h) * s.B + bt] = (float)sumB;
      }
    }
  }
}

// dA, ddt_bias: the sequences' sums in a fixed order, a block per value.
__global__ void __launch_bounds__(256) k_delta_fold_gates(const float* part, long B, int H, float* dA, float* dbias) {
  __shared__ double sh[256];
  const float* p = part + (long)blockIdx.x * B;
  double sum = 0.0;
  for (long i = threadIdx.x; i < B; i += 256) sum += (double)p[i];
  sh[threadIdx.x] = sum;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) sh[threadIdx.x] += sh[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x) return;
  if ((int)blockIdx.x < H) {
    if (dA) dA[blockIdx.x] = (float)sh[0];
  } else if (dbias) {
    dbias[blockIdx.x - H] = (float)sh[0];
  }
}
__global__ void __launch_bounds__(256) k_delta_zero_gates(int H, float* dA, float* dbias) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < H; i += gridDim.x * 256) {
    if (dA) dA[i] = 0.f;
    if (dbias) dbias[i] = 0.f;
  }
}

// dq and dk of shared heads: the value heads' in order, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) k_delta_fold_heads(const float* part, long rows, long B, int Hk, int H, int K, T* out,
                                                          long o_t, long o_b, long o_h) {
  const int rep = H / Hk;
  const long n = rows * Hk * K;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long row = i / ((long)Hk * K);
    const int e = (int)(i - row * Hk * K), hk = e / K, c = e % K;
    const float* p = part + (row * H + (long)hk * rep) * K + c;
    float sum = p[0];
    for (int r = 1; r < rep; r++) sum += p[(long)r * K];
    stf(out + row / B * o_t + row % B * o_b + hk * o_h + c, sum);
  }
}

// ---- single step ------------------------------------------------------------------------------------------
// Bound by the state, read and written once in fp32. A wavefront takes one head of one sequence and LPR * V of its columns: lane
// l the columns V (l % LPR) .. of the rows l / LPR, + 64 / LPR, ..., all in registers between the two passes over them.
template <typename T, int VEC, int LPR, int ROWS>
__global__ void __launch_bounds__(256) k_delta_step(const Args s, float* __restrict__ state, long items, int blocks_v) {
  constexpr int RG = 64 / LPR;
  static_assert(ROWS * RG <= 128, "rows of a state");
  __shared__ float sh[4][2][128];
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, cl = l % LPR, rg = l / LPR;
  for (long it = (long)blockIdx.x * 4 + w; it < items; it += (long)gridDim.x * 4) {
    const long unit_id = it / blocks_v, bt = unit_id / s.H;
    const int h = (int)(unit_id % s.H), hk = h / (s.H / s.Hk);
    const int c = (int)(it % blocks_v) * (LPR * VEC) + cl * VEC;
    const T* kp = (const T*)s.k + bt * s.k_b + hk * s.k_h;
    const T* qp = (const T*)s.q + bt * s.q_b + hk * s.q_h;
    float* sp = state + unit_id * (long)s.K * s.V + c;
    const bool fresh = s.first && s.first[bt] != 0.f;
    float x[ROWS][VEC];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int r = i * RG + rg;
#pragma unroll
      for (int j = 0; j < VEC; j++) x[i][j] = 0.f;
      if (r < s.K && c < s.V && !fresh) {
        if constexpr (VEC == 4) {
          const f4 v = *reinterpret_cast<const f4*>(sp + (long)r * s.V);
#pragma unroll
          for (int j = 0; j < VEC; j++) x[i][j] = v[j];
        } else {
          x[i][0] = sp[(long)r * s.V];
        }
      }
    }
    float kv[2], qv[2], kk = 0.f, qq = 0.f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int r = l + 64 * i;
      kv[i] = r < s.K ? ldf(kp + r) : 0.f;
      qv[i] = r < s.K ? ldf(qp + r) : 0.f;
      kk = fmaf(kv[i], kv[i], kk);
      qq = fmaf(qv[i], qv[i], qq);
    }
    group_sum<64>(kk, qq);
    const float rk = 1.f / sqrtf(kk + kEps), rq = 1.f / sqrtf(qq + kEps);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      sh[w][0][l + 64 * i] = kv[i] * rk;
      sh[w][1][l + 64 * i] = qv[i] * rq;
    }
    const float arg = ldf((const T*)s.a + bt * s.a_b + h) + (s.dt_bias ? s.dt_bias[h] : 0.f);
    const float al = ex2(log_decay(s.A[h], softplus(arg)) * (float)kLog2e);
    const float be = sigma(ldf((const T*)s.b + bt * s.b_b + h));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float e[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) e[j] = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const float kr = sh[w][0][i * RG + rg];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        x[i][j] *= al;
        e[j] = fmaf(x[i][j], kr, e[j]);
      }
    }
    float u[VEC], y[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
#pragma unroll
      for (int d = LPR; d < 64; d *= 2) e[j] += __shfl_xor(e[j], d);
      u[j] = c + j < s.V ? be * (ldf((const T*)s.v + bt * s.v_b + h * s.v_h + c + j) - e[j]) : 0.f;
      y[j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int r = i * RG + rg;
      const float kr = sh[w][0][r], qr = sh[w][1][r];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        x[i][j] = fmaf(kr, u[j], x[i][j]);
        y[j] = fmaf(x[i][j], qr, y[j]);
      }
      if (r < s.K && c < s.V) {
        if constexpr (VEC == 4) *reinterpret_cast<f4*>(sp + (long)r * s.V) = f4{x[i][0], x[i][1], x[i][2], x[i][3]};
        else sp[(long)r * s.V] = x[i][0];
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; j++) {
#pragma unroll
      for (int d = LPR; d < 64; d *= 2) y[j] += __shfl_xor(y[j], d);
      if (rg == 0 && c + j < s.V) stf((T*)s.y + bt * s.y_b + h * s.y_h + c + j, s.scale * y[j]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---- host ------------------------------------------------------------------------------------------
constexpr size_t kMaxDim = 128;
constexpr long kMaxBlocks = 1L << 20;  // a launch of 2^32 threads or more would not all start: blocks go on to their next units

int check(const ph_delta_args& p, const char* who) {
  PH_REQUIRE(p.dtype == PH_F32 || p.dtype == PH_BF16, "%s: dtype must be F32 or BF16", who);
  PH_REQUIRE(p.K >= 1 && p.K <= kMaxDim && p.V >= 1 && p.V <= kMaxDim, "%s: heads of K = %zu, V = %zu (at most 128)", who, p.K, p.V);
  PH_REQUIRE(p.Hk >= 1 && p.H >= p.Hk && p.H % p.Hk == 0 && p.H <= (1u << 16), "%s: %zu heads on %zu key heads", who, p.H, p.Hk);
  PH_REQUIRE(p.T <= (1u << 30) && p.B <= (1u << 24) && p.T * p.B <= (1ull << 40), "%s: T = %zu, B = %zu out of range", who, p.T, p.B);
  PH_REQUIRE(p.scale == p.scale, "%s: scale is not a number", who);
  if (p.T == 0 || p.B == 0) return PH_OK;
  PH_REQUIRE(p.q && p.k && p.v && p.a && p.b && p.A, "%s: q, k, v, a, b or A missing", who);
  return PH_OK;
}

bool rows_aligned(int dtype, const void* p, size_t width, long t, long b, long h) {
  const int v = dtype == PH_BF16 ? 8 : 4;
  return ((uintptr_t)p % 16) == 0 && width % v == 0 && t % v == 0 && b % v == 0 && h % v == 0;
}

Args args_of(const ph_delta_args& p) {
  Args a{};
  a.T = (long)p.T; a.B = (long)p.B; a.units = (long)(p.B * p.H);
  a.Hk = (int)p.Hk; a.H = (int)p.H; a.K = (int)p.K; a.V = (int)p.V;
  a.q = p.q; a.k = p.k; a.v = p.v; a.a = p.a; a.b = p.b;
  a.q_t = p.q_t; a.q_b = p.q_b; a.q_h = p.q_h; a.k_t = p.k_t; a.k_b = p.k_b; a.k_h = p.k_h;
  a.v_t = p.v_t; a.v_b = p.v_b; a.v_h = p.v_h; a.a_t = p.a_t; a.a_b = p.a_b; a.b_t = p.b_t; a.b_b = p.b_b;
  a.A = p.A; a.dt_bias = p.dt_bias; a.done = p.done; a.first = p.first; a.h0 = p.h0;
  a.scale = p.scale;
  a.vec = rows_aligned(p.dtype, p.q, p.K, p.q_t, p.q_b, p.q_h) && rows_aligned(p.dtype, p.k, p.K, p.k_t, p.k_b, p.k_h) &&
          rows_aligned(p.dtype, p.v, p.V, p.v_t, p.v_b, p.v_h);
  return a;
}

int padded(const Args& a) {
  const int d = a.K > a.V ? a.K : a.V;
  return d <= 32 ? 32 : d <= 64 ? 64 : 128;
}
unsigned blocks_of(long n) { return (unsigned)(n < kMaxBlocks ? n : kMaxBlocks); }

template <bool BF> int fwd_t(const Args& a, hipStream_t st) {
  const unsigned n = blocks_of(a.units);
  switch (padded(a)) {
    case 32: k_delta_fwd<BF, 32><<<n, 128, 0, st>>>(a); break;
    case 64: k_delta_fwd<BF, 64><<<n, 256, 0, st>>>(a); break;
    default: k_delta_fwd<BF, 128><<<n, 512, 0, st>>>(a);
  }
  PH_LAUNCH_CHECK();
  return PH_OK;
}

template <bool BF> int bwd_t(const Args& a, const GradArgs& o, float* dA, float* dbias, hipStream_t st) {
  using T = typename Elem<BF>::type;
  const unsigned n = blocks_of(a.units);
  switch (padded(a)) {
    case 32: k_delta_bwd<BF, 32><<<n, 128, 0, st>>>(a, o); break;
    case 64: k_delta_bwd<BF, 64><<<n, 256, 0, st>>>(a, o); break;
    default: k_delta_bwd<BF, 128><<<n, 512, 0, st>>>(a, o);
  }
  PH_LAUNCH_CHECK();
  if (o.gpart) {
    k_delta_fold_gates<<<2 * a.H, 256, 0, st>>>(o.gpart, a.B, a.H, dA, dbias);
    PH_LAUNCH_CHECK();
  }
  if (o.qpart) {
    const long e = a.T * a.B * a.Hk * a.K;
    const unsigned blocks = (unsigned)((e + 255) / 256 < 8192 ? (e + 255) / 256 : 8192);
    if (o.dq) k_delta_fold_heads<T><<<blocks, 256, 0, st>>>(o.qpart, a.T * a.B, a.B, a.Hk, a.H, a.K, (T*)o.dq, o.dq_t, o.dq_b, o.dq_h);
    if (o.dk) k_delta_fold_heads<T><<<blocks, 256, 0, st>>>(o.kpart, a.T * a.B, a.B, a.Hk, a.H, a.K, (T*)o.dk, o.dk_t, o.dk_b, o.dk_h);
    PH_LAUNCH_CHECK();
  }
  return PH_OK;
}

template <typename T, int VEC, int LPR> int step_rows(const Args& a, float* h, hipStream_t st) {
  constexpr int RG = 64 / LPR;
  const int blocks_v = (a.V + LPR * VEC - 1) / (LPR * VEC);
  const long items = a.units * blocks_v, blocks = (items + 3) / 4;
  const unsigned n = blocks_of(blocks);
  const int rows = (a.K + RG - 1) / RG;
  auto go = [&](auto r) { k_delta_step<T, VEC, LPR, decltype(r)::value><<<n, 256, 0, st>>>(a, h, items, blocks_v); };
  if (rows <= 8) {
    go(std::integral_constant<int, 8>());
  } else if (RG > 8 || rows <= 16) {
    go(std::integral_constant<int, 16>());
  } else if constexpr (RG <= 4) {
    if (RG == 4 || rows <= 32) {
      go(std::integral_constant<int, 32>());
    } else if constexpr (RG == 1) {
      if (rows <= 64) go(std::integral_constant<int, 64>());
      else go(std::integral_constant<int, 128>());
    }
  }
  PH_LAUNCH_CHECK();
  return PH_OK;
}
template <typename T> int step_t(const Args& a, float* h, hipStream_t st) {
  if (a.V % 4 == 0 && ((uintptr_t)h % 16) == 0) return a.V <= 32 ? step_rows<T, 4, 8>(a, h, st) : step_rows<T, 4, 16>(a, h, st);
  return a.V <= 16 ? step_rows<T, 1, 16>(a, h, st) : step_rows<T, 1, 64>(a, h, st);
}

long chunk_steps(int dtype) { return dtype == PH_BF16 ? Elem<true>::CH : Elem<false>::CH; }

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" size_t ph_delta_keep_floats(const ph_delta_args* p) {
  if (!p) return 0;
  const size_t c = (size_t)chunk_steps(p->dtype);
  return (p->T + c - 1) / c * p->B * p->H * p->K * p->V;
}

extern "C" int ph_delta_scan(const ph_delta_args* p, void* y, long y_t, long y_b, long y_h, float* h_out, float* keep,
                             void* stream) {
  PH_REQUIRE(p, "delta_scan: arguments missing");
  PH_TRY(check(*p, "delta_scan"));
  if (p->B == 0) return PH_OK;
  PH_REQUIRE(p->T >= 1, "delta_scan: no steps");
  PH_REQUIRE(y, "delta_scan: y missing");
  PH_REQUIRE(y != p->q && y != p->k && y != p->v, "delta_scan: y may not be q, k or v");
  Args a = args_of(*p);
  a.y = y; a.y_t = y_t; a.y_b = y_b; a.y_h = y_h; a.h_out = h_out; a.keep = keep;
  return p->dtype == PH_BF16 ? fwd_t<true>(a, as_stream(stream)) : fwd_t<false>(a, as_stream(stream));
}

extern "C" int ph_delta_scan_grad(const ph_delta_args* p, const float* keep, const void* dy, long dy_t, long dy_b, long dy_h,
                                  const float* dh, const ph_delta_grads* g, void* stream) {
  PH_REQUIRE(p && g, "delta_scan_grad: arguments missing");
  PH_TRY(check(*p, "delta_scan_grad"));
  hipStream_t st = as_stream(stream);
  if (p->B == 0) {  // no sequences: the parameters' sums are zero
    k_delta_zero_gates<<<64, 256, 0, st>>>((int)p->H, g->dA, g->ddt_bias);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  PH_REQUIRE(p->T >= 1, "delta_scan_grad: no steps");
  PH_REQUIRE(dy && keep, "delta_scan_grad: dy or the kept states missing");
  for (const void* out : {(const void*)g->dq, (const void*)g->dk, (const void*)g->dv})
    PH_REQUIRE(!out || (out != p->q && out != p->k && out != p->v && out != dy), "delta_scan_grad: a gradient may not be an input");
  Args a = args_of(*p);
  a.vec = a.vec && rows_aligned(p->dtype, dy, p->V, dy_t, dy_b, dy_h);
  GradArgs o{};
  o.dy = dy; o.dy_t = dy_t; o.dy_b = dy_b; o.dy_h = dy_h; o.keep = keep; o.dh = dh;
  o.dq = g->dq; o.dq_t = g->dq_t; o.dq_b = g->dq_b; o.dq_h = g->dq_h;
  o.dk = g->dk; o.dk_t = g->dk_t; o.dk_b = g->dk_b; o.dk_h = g->dk_h;
  o.dv = g->dv; o.dv_t = g->dv_t; o.dv_b = g->dv_b; o.dv_h = g->dv_h;
  o.da = g->da; o.da_t = g->da_t; o.da_b = g->da_b;
  o.db = g->db; o.db_t = g->db_t; o.db_b = g->db_b;
  o.dh0 = g->dh0;
  const bool shared = p->Hk != p->H && (g->dq || g->dk), gates = g->dA || g->ddt_bias;
  const size_t nq = shared ? p->T * p->B * p->H * p->K : 0, ng = gates ? 2 * p->H * p->B : 0;
  if (nq + ng) {
    float* ws = (float*)scratch(kSlotDelta, (2 * nq + ng) * 4);
    if (!ws) return PH_ERR_NOMEM;
    o.qpart = nq ? ws : nullptr;
    o.kpart = nq ? ws + nq : nullptr;
    o.gpart = ng ? ws + 2 * nq : nullptr;
  }
  return p->dtype == PH_BF16 ? bwd_t<true>(a, o, g->dA, g->ddt_bias, st) : bwd_t<false>(a, o, g->dA, g->ddt_bias, st);
}

extern "C" int ph_delta_step(const ph_delta_args* p, void* y, long y_b, long y_h, float* h, void* stream) {
  PH_REQUIRE(p, "delta_step: arguments missing");
  PH_REQUIRE(p->T <= 1, "delta_step: T = %zu (a single step)", p->T);
  PH_TRY(check(*p, "delta_step"));
  if (p->T == 0 || p->B == 0) return PH_OK;
  PH_REQUIRE(y && h, "delta_step: y or the state missing");
  PH_REQUIRE(y != p->q && y != p->k && y != p->v, "delta_step: y may not be q, k or v");
  Args a = args_of(*p);
  a.y = y; a.y_b = y_b; a.y_h = y_h;
  return p->dtype == PH_BF16 ? step_t<uint16_t>(a, h, as_stream(stream)) : step_t<float>(a, h, as_stream(stream));
}
