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
// state does not pass. Inside the products 0 times a non-finite value would; a chunk that finds one is done again in parts, with the
// other rows zero: episode by episode, and forward, where a step may not see the ones behind it, up to each step at which a column turns
// non-finite. (Backward every step sees the ones behind it.)
//
// Layout. A block owns one head of one sequence, wavefront w the state's columns 16 w .. 16 w + 15 (gradient: rows of the
// transposed state too), in the accumulator layout of the 16x16 matrix instructions: lane l holds rows 4 (l / 16) + r, column
// l % 16. That layout is also the one of the instruction's right operand when the contraction runs over
// those rows, so S, U and dY go from one product to the next without leaving the registers, and all of a wavefront's chain
// stays in its columns. bf16 rows enter the products as they are (their norms are factors outside). Values held in fp32 enter
// as sums of three bf16, all 24 bits, and the products of a chunk's small matrices and of the join are fp32 ones, so that what is not
// rounded to bf16 in the end is as precise as from fp32 inputs. fp32 takes the fp32 matrix instructions.
//
// Long sequences of few heads do not fill the chip, so time is cut into segments: a first launch runs each from a zero state and,
// without values, from the unit matrix, which gives what it adds to a state (Psi) and what it multiplies it with (Phi); a second
// joins the segments' start states in order; the third runs them again from those. The gradient does the same in reverse, with Phi^T.
//
// Measured, bf16: 64 steps of 2048 sequences x 8 heads of 64x64 forward with kept states 390 us (4.2 TB/s of what it moves; a large
// copy 5.2), gradient 1190 us: vector instructions issue for 44 % of it, matrix instructions for 22 %, two wavefronts on a SIMD wait at
// seven barriers a chunk for the rest (three wavefronts, with 168 registers, spill and took half as long again). With operands of
// two parts, 16 bits, in the gradient it was 1051 us, and dh0 off by 3e-6 of its norm where it is 2e-7. 2048 steps of 8 x 4 heads of
// 128x128 178 and 383 us; 8192 of 2 x 8 of 64x64 142 and 270 (in one piece 1575 and 4663 at first). A single step of 4096 x 8 heads of
// 64x64 195 us, 5.6 TB/s.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "routes.hpp"
#include "spans.hpp"

#include <type_traits>

namespace ph {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef u4 u4_any __attribute__((aligned(2)));  // 16 bytes at the alignment of an element
typedef f4 f4_any __attribute__((aligned(4)));

constexpr float kEps = 1e-6f;
constexpr double kLog2e = 1.4426950408889634;

struct Args {
  long T, B, units;  // units: sequences x heads
  int Hk, H, K, V;
  const void *q, *k, *v, *a, *b;
  long q_t, q_b, q_h, k_t, k_b, k_h, v_t, v_b, v_h, a_t, a_b, b_t, b_b;
  const float *A, *dt_bias, *done, *first, *h0;
  float scale;
  int segs;  // segments of time, of seg_chunks chunks each
  long seg_chunks;
  void* y;
  long y_t, y_b, y_h;
  float *h_out, *keep;
  float* start;  // [segs][units] states at the segments' starts (more than one segment)
  float *psi, *phi;  // [segs][units]: what a segment adds to its start state, and what it multiplies it with (parts = 2: tiles transposed)
  int* cut;          // [segs][units]: an episode starts in the segment, and nothing passes it
  int local_from, parts;  // of these: segments from local_from on, segs - 1 of them; both, or phi alone
};

struct GradArgs {
  const void* dy;
  long dy_t, dy_b, dy_h;
  const float *keep, *dh;
  void *dq, *dk, *dv, *da, *db;
  long dq_t, dq_b, dq_h, dk_t, dk_b, dk_h, dv_t, dv_b, dv_h, da_t, da_b, db_t, db_b;
  float* dh0;
  float *qpart, *kpart;  // [T][B][H][K] of every value head, where heads share their keys
  float* gpart;          // [2][H][segs B]: sums of dlog al softplus and of dlog al A sigmoid
  float *dend, *xi;      // [segs][units] gradients of the segments' end states; [segs][units] what a segment adds on the way back
};

// The kernel's own arguments, read again from where the launch put them: Args first, GradArgs behind. The compiler reads
// arguments once, at the kernel's start, and what the scalar registers cannot hold over the loops it keeps in lanes of
// vector registers.
template <typename A> __device__ __forceinline__ A again(unsigned at) {
  static_assert(sizeof(A) % 8 == 0 && alignof(A) == 8, "read in words of eight bytes");
  auto p = (const __attribute__((address_space(4))) uint64_t*)__builtin_amdgcn_kernarg_segment_ptr();
  asm("" : "+s"(p));
  uint64_t w[sizeof(A) / 8];
#pragma unroll
  for (unsigned i = 0; i < sizeof(A) / 8; i++) w[i] = p[at / 8 + i];
  return __builtin_bit_cast(A, w);
}

// Global pointers as such: of one that `again` has read the compiler does not know that it is none to LDS.
#define PH_GLOBAL __attribute__((address_space(1)))
template <typename T> using gin = const PH_GLOBAL T*;
template <typename T> using gout = PH_GLOBAL T*;

// ---- elements ------------------------------------------------------------------------------------------
__device__ __forceinline__ float ldf(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float ldf(gin<uint16_t> p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float ldf(gin<float> p) { return *p; }
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float raw_f32(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float raw_f32(float v) { return v; }
__device__ __forceinline__ void stf(uint16_t* p, float v) { *p = bf16_rne(v); }
__device__ __forceinline__ void stf(gout<uint16_t> p, float v) { *p = bf16_rne(v); }
__device__ __forceinline__ void stf(gout<float> p, float v) { *p = v; }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ float ex2(float v) { return __builtin_amdgcn_exp2f(v); }
// softplus, max(v, 0) + log(1 + e) with e = exp(-|v|). What rounding 1 + e to w dropped is added back as it is, so small e
// keep their digits.
__device__ __forceinline__ float softplus(float v) {
  const float e = ex2(-fabsf(v) * (float)kLog2e), w = 1.f + e;
  return fmaxf(v, 0.f) + fmaf(__builtin_amdgcn_logf(w), (float)(1 / kLog2e), e - (w - 1.f));
}
__device__ __forceinline__ float sigma(float v) { return __builtin_amdgcn_rcpf(1.f + ex2(v * -(float)kLog2e)); }
// max and comparisons with a NaN drop it; a gate of NaN stays one
__device__ __forceinline__ float log_decay(float A, float sp) {
  const float g = A * sp;
  return g < -1e9f ? -1e9f : g;  // differences of sums stay numbers
}
// Sums of a chunk's values below this are finite.
constexpr float kFar = 0x1p100f;

// From here on the compiler takes the lane's number as new: what depends on it alone is formed where it is used and does not wait
// in registers over all chunks.
__device__ __forceinline__ void renew(int& tid, int& l) {
  asm volatile("" : "+v"(tid));
  l = tid & 63;
}

// ---- matrix operands -------------------------------------------------------------------------------------
// Operands are taken in units of 16 of the contraction, of which lane l holds 4 (l / 16) + 0..3.
template <bool BF> struct Elem { using type = uint16_t; using unit = s4; static constexpr int CH = 32, pad = 8, V = 8; };
template <> struct Elem<false> { using type = float; using unit = f4; static constexpr int CH = 16, pad = 4, V = 4; };

// acc += a b over N units; bf16 units go in pairs.
template <int N> __device__ __forceinline__ f4 dot(const s4* a, const s4* b, f4 acc) {
  static_assert(N % 2 == 0, "whole pairs");
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const s8 x = __builtin_shufflevector(a[i], a[i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    const s8 y = __builtin_shufflevector(b[i], b[i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), acc, 0, 0, 0);
  }
  return acc;
}
template <int N> __device__ __forceinline__ f4 dot(const f4* a, const f4* b, f4 acc) {
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][r], b[i][r], acc, 0, 0, 0);
  return acc;
}

// fp32 values as operands: for bf16 three parts, each the nearest bf16 to what the ones before leave (24 bits, all there are), else
// the values themselves.
template <bool BF> struct Parts {
  s4 hi, mid, low;
  __device__ __forceinline__ void set(f4 v) {
    hi = nearest(v);
    mid = nearest(v);
    low = nearest(v);
  }
  __device__ __forceinline__ f4 sum() const { return (wide(low) + wide(mid)) + wide(hi); }

 private:
  static __device__ __forceinline__ f4 wide(s4 p) {
    const u2 u = __builtin_bit_cast(u2, p);
    return f4{__builtin_bit_cast(float, u[0] << 16), __builtin_bit_cast(float, u[0] & 0xffff0000u), __builtin_bit_cast(float, u[1] << 16),
              __builtin_bit_cast(float, u[1] & 0xffff0000u)};
  }
  static __device__ __forceinline__ s4 nearest(f4& v) {  // and what it leaves of v
    const s4 p = __builtin_bit_cast(s4, u2{bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3])});
    v -= wide(p);
    return p;
  }
};
template <> struct Parts<false> {
  f4 hi;
  __device__ __forceinline__ void set(f4 v) { hi = v; }
  __device__ __forceinline__ f4 sum() const { return hi; }
};
// acc += a b, the smallest products first: a exact rows and b in parts, and both in parts (products below 2^-24 of the largest
// are left out).
template <bool BF, int N>
__device__ __forceinline__ f4 dot_parts(const typename Elem<BF>::unit* a, const Parts<BF>* b, f4 acc) {
  typename Elem<BF>::unit h[N];
  if constexpr (BF) {
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = b[i].low;
    acc = dot<N>(a, h, acc);
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = b[i].mid;
    acc = dot<N>(a, h, acc);
  }
#pragma unroll
  for (int i = 0; i < N; i++) h[i] = b[i].hi;
  return dot<N>(a, h, acc);
}
template <bool BF, int N> __device__ __forceinline__ f4 dot_parts(const Parts<BF>* a, const Parts<BF>* b, f4 acc) {
  typename Elem<BF>::unit h[N];
  if constexpr (BF) {
    typename Elem<BF>::unit g[N];
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = a[i].low, g[i] = b[i].hi;
    acc = dot<N>(h, g, acc);
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = a[i].mid, g[i] = b[i].mid;
    acc = dot<N>(h, g, acc);
#pragma unroll
    for (int i = 0; i < N; i++) g[i] = b[i].hi;
    acc = dot<N>(h, g, acc);
  }
#pragma unroll
  for (int i = 0; i < N; i++) h[i] = a[i].hi;
  return dot_parts<BF, N>(h, b, acc);
}

// Units of a matrix in LDS, leading dimension LD. row_unit: row `row` + l % 16, columns `col` + 4 (l / 16) + 0..3 (left
// operand with the contraction over columns, or the right one of the transposed matrix); col_unit: rows `row` + 4 (l / 16) +
// 0..3, column `col` + l % 16 (contraction over rows), for 16-bit elements by the transposing load, which gives lane l of
// sixteen the column l of the four rows that the sixteen lanes' addresses cover.
template <int LD> __device__ __forceinline__ s4 row_unit(int tid, const uint16_t* m, int row, int col) {
  const int l = tid & 63;
  return *reinterpret_cast<const s4*>(m + (row + (l & 15)) * LD + col + 4 * (l >> 4));
}
template <int LD> __device__ __forceinline__ f4 row_unit(int tid, const float* m, int row, int col) {
  const int l = tid & 63;
  return *reinterpret_cast<const f4*>(m + (row + (l & 15)) * LD + col + 4 * (l >> 4));
}
template <int LD> __device__ __forceinline__ s4 col_unit(int tid, const uint16_t* m, int row, int col) {
  const int l = tid & 63;
  const uint16_t* p = m + (row + 4 * (l >> 4) + ((l & 15) >> 2)) * LD + col + 4 * (l & 3);
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
}
template <int LD> __device__ __forceinline__ f4 col_unit(int tid, const float* m, int row, int col) {
  const int l = tid & 63;
  const float* p = m + (row + 4 * (l >> 4)) * LD + col + (l & 15);
  return f4{p[0], p[LD], p[2 * LD], p[3 * LD]};
}
__device__ __forceinline__ f4 widen(s4 v) {
  return f4{bf16_to_f32((uint16_t)v[0]), bf16_to_f32((uint16_t)v[1]), bf16_to_f32((uint16_t)v[2]), bf16_to_f32((uint16_t)v[3])};
}
__device__ __forceinline__ f4 widen(f4 v) { return v; }

// ---- a chunk's rows ------------------------------------------------------------------------------------
// The 16 bytes of a row of W columns that a thread stages: row tid / (P / V), columns from V (tid % (P / V)) on, at p; zero
// where the rows or the columns end. Any alignment: the hardware takes 16 bytes at that of an element. The last columns of a row
// come from an access that ends with it, shifted down.
template <bool BF, int P, typename T = typename Elem<BF>::type>
__device__ __forceinline__ u4 load_row(int tid, gin<T> p, int rows, int W) {
  constexpr int V = Elem<BF>::V;
  const int row = tid / (P / V), c = tid % (P / V) * V;
  if (rows == Elem<BF>::CH && W == P) return *(gin<u4_any>)p;
  u4 r = {0, 0, 0, 0};
  if (row < rows && c < W) {
    const int over = c + V - W;
    if (W >= V) {
      const int skip = over > 0 ? over : 0;
      r = *(gin<u4_any>)(p - skip);
      if (over > 0) r = __builtin_bit_cast(u4, __builtin_bit_cast(unsigned __int128, r) >> (skip * 8 * (int)sizeof(T)));
    } else {
      unsigned __int128 x = 0;
#pragma unroll 1
      for (int i = W - 1; i >= 0; i--) x = x << (8 * (int)sizeof(T)) | (sizeof(T) == 2 ? (unsigned)*(gin<uint16_t>)(p + i) : *(gin<unsigned>)(p + i));
      r = __builtin_bit_cast(u4, x);
    }
  }
  return r;
}
// The first n of 16 bytes' elements from LDS to a row.
template <bool BF, typename T = typename Elem<BF>::type> __device__ __forceinline__ void store_row(gout<T> p, const T* from, int n) {
  constexpr int V = Elem<BF>::V;
  if (n >= V) {
    *(gout<u4_any>)p = *reinterpret_cast<const u4*>(from);
  } else {
#pragma unroll 1
    for (int i = 0; i < n; i++) p[i] = from[i];
  }
}
template <bool BF, int P, typename T> __device__ __forceinline__ gin<T> thread_row(int tid, const T* base, long stride, long t0) {
  constexpr int V = Elem<BF>::V;
  return (gin<T>)base + (t0 + tid / (P / V)) * stride + tid % (P / V) * V;
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
// All below kFar.
template <bool BF> __device__ __forceinline__ bool all_near(u4 r) {
  constexpr uint32_t far = __builtin_bit_cast(uint32_t, kFar);
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t u = r[i];
    if constexpr (BF) ok = ok && (u & 0x7f80u) < far >> 16;
    ok = ok && (u & 0x7f800000u) < far;
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
  float c0;                           // D_c0
  int starts;                         // bit i: row i starts an episode
  int odd, split;                     // what mark_odd has found
};

// The lane's row of the gates, loaded ahead: as it is in memory, for what is computed from it would be waited for.
template <typename T> struct Gate {
  T a, b;
  float bias, start;
};
template <typename T> __device__ __forceinline__ Gate<T> load_gate(long bt, int h, long t0, int rows, int i) {
  Gate<T> g = {T(0), T(0), 0.f, 0.f};
  const Args s = again<Args>(0);
  if (i < rows) {
    const long t = t0 + i;
    g.a = *((gin<T>)s.a + t * s.a_t + bt * s.a_b + h);
    g.b = *((gin<T>)s.b + t * s.b_t + bt * s.b_b + h);
    if (s.dt_bias) g.bias = ((gin<float>)s.dt_bias)[h];
    gin<float> f = (gin<float>)(t > 0 ? s.done : s.first);
    if (f) g.start = f[t > 0 ? (t - 1) * s.B + bt : bt];
  }
  return g;
}
template <int CTL> __device__ __forceinline__ double dpp_f64(double v) {  // zero where the shift leaves the row of lanes
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float lane_f32(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// Fills r for rows lo..hi-1 from the gates in a wavefront's lanes (all of it calls), but for the norms.
template <int CH, typename T> __device__ __forceinline__ void fill_rows(int tid, Rows<CH>& r, const Gate<T>& g, float A, int lo, int hi) {
  const int i = tid & 63;
  const bool in = i >= lo && i < hi;
  const float arg = raw_f32(g.a) + g.bias, sp = softplus(arg);
  double G = in ? (double)log_decay(A, sp) * kLog2e : 0.0;
  const unsigned long long starts = __ballot(in && g.start != 0.f);
  G += dpp_f64<0x111>(G);  // sums along the rows of 16 lanes
  G += dpp_f64<0x112>(G);
  G += dpp_f64<0x114>(G);
  G += dpp_f64<0x118>(G);
  if constexpr (CH == 32) {
    const double low = lane_f64(G, 15);
    if (i & 16) G += low;
  }
  const double last = lane_f64(G, CH - 1);
  const float be = in ? sigma(raw_f32(g.b)) : 0.f;
  const bool none = __any(!(be <= 1.f) || G != G);
  if (i < CH) {
    const int seg = __popcll(starts & ((2ull << i) - 1)), all = __popcll(starts);
    r.G[i] = G;
    r.seg[i] = seg;
    r.be[i] = be;
    r.sp[i] = sp;
    r.arg[i] = arg;
    const float d0 = ex2((float)G), dc = ex2((float)(last - G));
    r.d0[i] = in && (seg == 0 || d0 != d0) ? d0 : 0.f;  // a gate that is none shows in Y also behind an episode's start
    r.dc[i] = in && seg == all ? dc : 0.f;
    if (i == CH - 1) {
      r.c0 = all == 0 ? d0 : 0.f;
      r.starts = (int)(starts & 0xffffffffu);
      r.odd = none || last > 40.0;  // a decay that grows (A above 0) may pass fp32's range in M, which Y does not show
      r.split = CH;
    }
  }
}
// Rows lo..hi-1 of a wavefront's columns of Y that are not finite (nor far enough from the largest number for sums of them to be): that there
// are any, and the first one that has a row in front of it in its column. Those in front may not meet it in a product; behind it all of
// the column's are none either.
template <int CH, int NB> __device__ __forceinline__ void mark_odd(int tid, Rows<CH>& r, const f4* Y, int lo, int hi) {
  bool odd = false;
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int i = 0; i < 4; i++) odd |= !(fabsf(Y[n][i]) < kFar);
  if (!__any(odd)) return;
  const int l = tid & 63;
  unsigned rows = 0;
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int i = 0; i < 4; i++) rows |= !(fabsf(Y[n][i]) < kFar) ? 1u << (16 * n + 4 * (l >> 4) + i) : 0u;
  rows |= (unsigned)__shfl_xor((int)rows, 16);
  rows |= (unsigned)__shfl_xor((int)rows, 32);
  rows &= (2u << (hi - 1)) - (1u << lo);
  if (!rows) return;
  r.odd = 1;
  const int at = __ffs((int)rows) - 1;
  if (at > lo) atomicMin(&r.split, at);
}
__device__ __forceinline__ f4 rows4(int tid, const float* r, int at) { return *reinterpret_cast<const f4*>(r + at + 4 * ((tid & 63) >> 4)); }

// Small matrices of a chunk are kept transposed, in fp32: a tile's lane holds four rows of a column, one access of them. Their
// products are fp32 ones: few, and fp32 saves cutting their operands in parts.
template <int N> struct alignas(16) Mat {
  float v[N];
};
template <int LD, int N> __device__ __forceinline__ void put_mat(int tid, Mat<N>& m, int row, int col, f4 v) {
  const int l = tid & 63;
  *reinterpret_cast<f4*>(m.v + (row + (l & 15)) * LD + col + 4 * (l >> 4)) = v;
}
// The left operand of the matrix itself (tile's row `row`, column `col` of the stored, transposed one) and of its transpose, which is
// also the four values that put_mat of the same place took.
template <int LD, int N> __device__ __forceinline__ f4 mat_col(int tid, const Mat<N>& m, int row, int col) {
  return col_unit<LD>(tid, m.v, row, col);
}
template <int LD, int N> __device__ __forceinline__ f4 mat_row(int tid, const Mat<N>& m, int row, int col) {
  return row_unit<LD>(tid, m.v, row, col);
}

// A chunk's M, P and T = (I + M)^-1. Of T the diagonal blocks; of M these also as they are, for the substitution.
template <bool BF, bool WITH_P> struct Scores {
  static constexpr int CH = Elem<BF>::CH, UD = CH + 4, TD = 20;
  Mat<CH * UD> M;
  Mat<WITH_P ? CH * UD : 1> P;
  Mat<CH * TD> Tinv;
};

// M (and P) of the chunk: tiles on and below the diagonal, dealt out over the wavefronts.
template <bool BF, int P, int LD, bool WITH_P, int NM, int NP>
__device__ __forceinline__ void score_tiles(int tid, const Rows<Elem<BF>::CH>& r, const typename Elem<BF>::type* Qs,
                                            const typename Elem<BF>::type* Ks, Mat<NM>& M, Mat<NP>& Pm, float* diag, float scale) {
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, NT = P / 16, UD = CH + 4, TILES = NB * (NB + 1) / 2;
  const int l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int id = w; id < (WITH_P ? 2 : 1) * TILES; id += NT) {
    const bool isP = WITH_P && id >= TILES;
    const int tile = isP ? id - TILES : id, bi = tile == 0 ? 0 : 1, bj = tile == 2 ? 1 : 0;  // (0,0) (1,0) (1,1)
    typename Elem<BF>::unit x[NT], y[NT];
#pragma unroll
    for (int m = 0; m < NT; m++) {
      x[m] = row_unit<LD>(tid, isP ? Qs : Ks, 16 * bi, 16 * m);
      y[m] = row_unit<LD>(tid, Ks, 16 * bj, 16 * m);
    }
    f4 acc = dot<NT>(x, y, f4{0.f, 0.f, 0.f, 0.f});
    const int j = l & 15, i0 = 4 * (l >> 4);
    const double Gj = r.G[16 * bj + j];
    const int segj = r.seg[16 * bj + j];
    const float rkj = r.rk[16 * bj + j];
    const f4 ci = isP ? scale * rows4(tid, r.rq, 16 * bi) : rows4(tid, r.be, 16 * bi) * rows4(tid, r.rk, 16 * bi);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int i = 16 * bi + i0 + k;
      const bool on = segj == r.seg[i] && (bi != bj || (isP ? j <= i0 + k : j < i0 + k));
      acc[k] = on ? ex2((float)(r.G[i] - Gj)) * rkj * ci[k] * acc[k] : 0.f;
    }
    if constexpr (WITH_P) {
      if (isP) {
        put_mat<UD>(tid, Pm, 16 * bj, 16 * bi, acc);
        continue;
      }
    }
    put_mat<UD>(tid, M, 16 * bj, 16 * bi, acc);
    if (bi == bj) {
#pragma unroll
      for (int k = 0; k < 4; k++) diag[(16 * bi + i0 + k) * 16 + j] = acc[k];
    }
  }
}

// The diagonal blocks of (I + M)^-1, one column per lane of a wavefront's first CH.
template <int CH, int N> __device__ __forceinline__ void invert_blocks(int tid, const float* diag, Mat<N>& Tinv) {
  const int l = tid & 63;
  if (l >= CH) return;
  const int o = l & ~15, c = l & 15;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    float s = i == c ? 1.f : 0.f;
#pragma unroll
    for (int j4 = 0; j4 < i; j4 += 4) {
      const f4 m = *reinterpret_cast<const f4*>(diag + (o + i) * 16 + j4);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (j4 + k < i) s = fmaf(-m[k], x[j4 + k], s);
    }
    x[i] = s;
  }
#pragma unroll
  for (int i = 0; i < 16; i += 4) *reinterpret_cast<f4*>(Tinv.v + l * 20 + i) = f4{x[i], x[i + 1], x[i + 2], x[i + 3]};
}

// U = T Y by blocks, T's blocks below the diagonal through M.
template <bool BF, int NM, int NI> __device__ __forceinline__ void solve(int tid, const Mat<NI>& Tinv, const Mat<NM>& M, const f4* Y, f4* U) {
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, UD = CH + 4;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 t = mat_col<20>(tid, Tinv, 0, 0);
  U[0] = dot<1>(&t, Y, zero);
  if constexpr (NB == 2) {
    f4 y = -U[0];
    t = mat_col<UD>(tid, M, 0, 16);
    y = dot<1>(&t, &y, Y[1]);
    t = mat_col<20>(tid, Tinv, 16, 0);
    U[1] = dot<1>(&t, &y, zero);
  }
}
// dY = T^T dU
template <bool BF, int NM, int NI> __device__ __forceinline__ void solve_t(int tid, const Mat<NI>& Tinv, const Mat<NM>& M, const f4* dU, f4* dY) {
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, UD = CH + 4;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  f4 top = dU[0], t;
  if constexpr (NB == 2) {
    t = mat_row<20>(tid, Tinv, 16, 0);
    dY[1] = dot<1>(&t, dU + 1, zero);
    const f4 y = -dY[1];
    t = mat_row<UD>(tid, M, 0, 16);
    top += dot<1>(&t, &y, zero);
  }
  t = mat_row<20>(tid, Tinv, 0, 0);
  dY[0] = dot<1>(&t, &top, zero);
}

// States in memory: [K][V] as the caller holds them; the library's own in whole tiles of 16x16, [K tiles][V tiles], each as the
// lanes hold it: lane l's four rows 4 (l / 16) + 0..3 of column l % 16.
__host__ __device__ __forceinline__ int up16(int n) { return (n + 15) & ~15; }
struct Own {
  int tk, tv;  // tiles
  __device__ __forceinline__ long floats() const { return (long)tk * tv * 256; }
};
// Tile m of column block w; one past the last is taken as the last: its rows meet keys and queries of zero.
__device__ __forceinline__ f4 own_tile(int tid, gin<float> s, Own d, int m, int w) {
  const int tile = (m < d.tk ? m : d.tk - 1) * d.tv + (w < d.tv ? w : d.tv - 1);
  return *reinterpret_cast<gin<f4>>(s + tile * 256 + 4 * (tid & 63));
}
// The transposed state's tile m of block w: columns of V 16 m + 4 (l / 16) + 0..3, row 16 w + l % 16.
__device__ __forceinline__ f4 own_tile_t(int tid, gin<float> s, Own d, int m, int w) {
  const int l = tid & 63, tile = (w < d.tk ? w : d.tk - 1) * d.tv + (m < d.tv ? m : d.tv - 1);
  gin<float> p = s + tile * 256 + ((l >> 2 & 3) * 16 + 4 * (l >> 4)) * 4 + (l & 3);
  return f4{p[0], p[4], p[8], p[12]};
}
__device__ __forceinline__ void put_own_tile(int tid, gout<float> s, Own d, int m, int w, f4 x) {
  if (m < d.tk && w < d.tv) *reinterpret_cast<gout<f4>>(s + (m * d.tv + w) * 256 + 4 * (tid & 63)) = x;
}
// The same into a matrix whose tiles lie transposed: there a lane's four values are columns 4 (l / 16) + 0..3 of row l % 16.
__device__ __forceinline__ void put_own_tile_t(int tid, gout<float> s, Own d, int m, int w, f4 x) {
  const int l = tid & 63;
  gout<float> p = s + (m * d.tv + w) * 256 + (4 * (l >> 4) + 16 * (l >> 2 & 3)) * 4 + (l & 3);
  if (m < d.tk && w < d.tv) p[0] = x[0], p[4] = x[1], p[8] = x[2], p[12] = x[3];
}
// All tiles of column block w of a caller's state, or (T) of the transposed one's; zero outside. Addresses are clamped and not
// skipped: a load that a branch guards is waited for before the next one.
template <int NT, bool TR> __device__ __forceinline__ void get_state(int tid, gin<float> s, int K, int V, int w, f4* S) {
  const int l = tid & 63, in = l & 15, four = 4 * (l >> 4);
  if (((K | V) & 15) == 0) {
#pragma unroll
    for (int m = 0; m < NT; m++) {
      S[m] = f4{0.f, 0.f, 0.f, 0.f};
      if (16 * m < (TR ? V : K) && 16 * w < (TR ? K : V)) {
        if constexpr (TR) {
          S[m] = *(gin<f4_any>)(s + (16 * w + in) * V + 16 * m + four);
        } else {
          const unsigned at = (four * V + in) * 4;
#pragma unroll
          for (int i = 0; i < 4; i++) S[m][i] = *(gin<float>)((gin<char>)(s + (16 * m + i) * V + 16 * w) + at);
        }
      }
    }
    return;
  }
#pragma unroll 1
  for (int m = 0; m < NT; m++) {
    f4 x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int k = TR ? 16 * w + in : 16 * m + four + i, v = TR ? 16 * m + four + i : 16 * w + in;
      const float y = s[k < K && v < V ? k * V + v : 0];
      x[i] = k < K && v < V ? y : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NT; j++) S[j] = j == m ? x : S[j];
  }
}
template <int NT> __device__ __forceinline__ void put_state(int tid, gout<float> s, int K, int V, int w, const f4* S) {
  const int l = tid & 63, c = 16 * w + (l & 15), four = 4 * (l >> 4);
  if (((K | V) & 15) == 0) {
    const unsigned at = (four * V + (l & 15)) * 4;
    if (16 * w < V) {
#pragma unroll
      for (int m = 0; m < NT; m++)
        if (16 * m < K) {
#pragma unroll
          for (int i = 0; i < 4; i++) *(gout<float>)((gout<char>)(s + (16 * m + i) * V + 16 * w) + at) = S[m][i];
        }
    }
    return;
  }
  if (c >= V) return;
#pragma unroll
  for (int m = 0; m < NT; m++) {
    gout<float> p = s + (16 * m + four) * V + c;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (16 * m + four + i < K) p[i * V] = S[m][i];
  }
}

template <bool BF, int P, typename T = typename Elem<BF>::type>
__device__ __forceinline__ void put_row(int tid, T* tile, u4 r, int lo, int hi, bool part) {
  constexpr int V = Elem<BF>::V, LD = P + Elem<BF>::pad;
  const int row = tid / (P / V), c = tid % (P / V) * V;
  if (part && (row < lo || row >= hi)) r = u4{0, 0, 0, 0};
  *reinterpret_cast<u4*>(tile + row * LD + c) = r;
}
// 1 / sqrt(|row|^2 + eps) of the staged rows, 0 for those left out, NaN for rows longer than fp32 can say, whose products are no
// numbers either. Returns whether the thread's row is such a one, or holds what is not finite.
template <bool BF, int P> __device__ __forceinline__ bool put_norm(int tid, float* out, u4 r, int lo, int hi) {
  constexpr int L = P / Elem<BF>::V;  // lanes of a row
  float s = square_sum<BF>(r);
  s += dpp_mov<0xB1>(s);
  s += dpp_mov<0x4E>(s);
  if constexpr (L >= 8) s += dpp_mov<0x141>(s);
  if constexpr (L >= 16) s += dpp_mov<0x140>(s);
  if constexpr (L >= 32) s += __shfl_xor(s, 16);
  const int row = tid / L;
  const bool in = row >= lo && row < hi, odd = in && !(s < INFINITY);
  if (tid % L == 0) out[row] = odd ? NAN : in ? __builtin_amdgcn_rsqf(s + kEps) : 0.f;
  return odd;
}

// ---- sequences ------------------------------------------------------------------------------------------
// Wavefronts of a SIMD, at least: as many as registers and LDS leave room for (three in the 64-wide fp32 gradient, 16 registers of it
// spilled: 64 steps of 512 x 8 heads 400 us, 467 with two and none spilled).
template <bool BF, int P> constexpr int fwd_waves() { return P == 128 ? 2 : BF && P == 32 ? 3 : 4; }
template <bool BF, int P> constexpr int bwd_waves() { return BF || P == 128 ? 2 : 3; }

// One segment of one sequence's head. LOCAL: without outputs, from a zero state (what the segment adds to its start state) or,
// without values to write, from the unit matrix (what it multiplies it with).
template <bool BF, int P, bool LOCAL> __global__ void __launch_bounds__(4 * P, (fwd_waves<BF, P>())) k_delta_fwd(const Args args) {
  using T = typename Elem<BF>::type;
  using unit = typename Elem<BF>::unit;
  constexpr int CH = Elem<BF>::CH, NB = CH / 16, NT = P / 16, LD = P + Elem<BF>::pad, UD = CH + 4;
  __shared__ __attribute__((aligned(16))) T Qs[LOCAL ? 1 : CH * LD], Ks[CH * LD], Vs[CH * LD];
  __shared__ __attribute__((aligned(16))) Scores<BF, !LOCAL> X;
  __shared__ __attribute__((aligned(16))) float diag[CH * 16];
  __shared__ Rows<CH> Rs[2];
  int tid = threadIdx.x, l = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  for (long item = blockIdx.x;; item += gridDim.x) {
    const Args s = again<Args>(0);
    if (item >= s.units * (LOCAL ? (s.segs - 1) * s.parts : s.segs)) break;
    const unsigned units = (unsigned)s.units, round = (unsigned)item / units;
    const long unit_id = (unsigned)item - round * units;
    const int part = LOCAL ? (s.parts == 1 ? 1 : (int)round & 1) : 0;
    const long seg = LOCAL ? (s.parts == 1 ? round : round >> 1) + s.local_from : round;
    const long bt = (unsigned)unit_id / (unsigned)s.H;
    const int h = (int)(unit_id - bt * s.H), hk = (int)((unsigned)h / (unsigned)(s.H / s.Hk));
    const Own own = {up16(s.K) / 16, up16(part ? s.K : s.V) / 16};
    const long first = seg * s.seg_chunks * CH;
    const long last = first + s.seg_chunks * CH < s.T ? first + s.seg_chunks * CH : s.T;
    gin<T> qp = thread_row<BF, P>(tid, (const T*)s.q + bt * s.q_b + hk * s.q_h, s.q_t, first);
    gin<T> kp = thread_row<BF, P>(tid, (const T*)s.k + bt * s.k_b + hk * s.k_h, s.k_t, first);
    gin<T> vp = thread_row<BF, P>(tid, (const T*)s.v + bt * s.v_b + h * s.v_h, s.v_t, first);
    const float A = s.A[h], scale = s.scale;
    auto rows_at = [&](long t0) { return (int)(t0 >= last ? 0 : last - t0 < CH ? last - t0 : CH); };
    f4 S[NT];
    if (LOCAL) {
#pragma unroll
      for (int m = 0; m < NT; m++) {
        S[m] = zero;
        if (part && m == w) {
#pragma unroll
          for (int i = 0; i < 4; i++) S[m][i] = 4 * (l >> 4) + i == (l & 15) ? 1.f : 0.f;
        }
      }
    } else if (s.segs > 1) {
#pragma unroll
      for (int m = 0; m < NT; m++) {
        S[m] = own_tile(tid, (gin<float>)s.start + (seg * s.units + unit_id) * own.floats(), own, m, w);
        if (m >= own.tk || w >= own.tv) S[m] = zero;
      }
    } else if (s.h0) {
      get_state<NT, false>(tid, (gin<float>)s.h0 + unit_id * s.K * s.V, s.K, s.V, w, S);
    } else {
#pragma unroll
      for (int m = 0; m < NT; m++) S[m] = zero;
    }
    int rows = rows_at(first);
    u4 q = {0, 0, 0, 0}, k, v;
    auto load = [&]() {
      const Args a = again<Args>(0);
      if (!LOCAL) q = load_row<BF, P>(tid, qp, rows, a.K);
      k = load_row<BF, P>(tid, kp, rows, a.K);
      v = load_row<BF, P>(tid, vp, rows, part ? 0 : a.V);
    };
    auto walk = [&](int chunks) {
      const Args a = again<Args>(0);
      qp += chunks * CH * a.q_t;
      kp += chunks * CH * a.k_t;
      vp += chunks * CH * a.v_t;
    };
    bool have = false;  // this chunk's rows are there
    // the last wavefront sees to the gates, a chunk ahead
    Gate<T> g = {}, gn = g;
    if (w == NT - 1) {
      g = load_gate<T>(bt, h, first, rows, l);
      gn = load_gate<T>(bt, h, first + CH, rows_at(first + CH), l);
    }
    __syncthreads();  // the item before has been read
    if (w == NT - 1) fill_rows<CH>(tid, Rs[0], g, A, 0, rows);
    int cur = 0, cut = 0, y_lo = 0, y_hi = 0;
    long y_at = first;
    auto put_y = [&](long at, int lo, int hi) {  // a thread stores the 16 bytes that it stages next
      const Args a = again<Args>(0);
      const int row = tid / (P / Elem<BF>::V), c = tid % (P / Elem<BF>::V) * Elem<BF>::V;
      if (row >= lo && row < hi)
        store_row<BF>((gout<T>)a.y + bt * a.y_b + h * a.y_h + (at + row) * a.y_t + c, Vs + row * LD + c, a.V - c);
    };
    for (long t0 = first; t0 < last; t0 += CH) {
      Rows<CH>& R = Rs[cur];
      if (!LOCAL) {
        const Args a = again<Args>(0);
        if (a.keep) {
          gout<float> to = (gout<float>)a.keep + (t0 / CH * a.units + unit_id) * own.floats();
#pragma unroll
          for (int m = 0; m < NT; m++) put_own_tile(tid, to, own, m, w, S[m]);
        }
      }
      const int all = rows;  // rows of this chunk
      for (int lo = 0, hi = all, once = 1; lo < all; once = 0) {
        __syncthreads();  // the rows before have been read
        renew(tid, l);
        if (!LOCAL) {
          put_y(y_at, y_lo, y_hi);
          y_hi = 0;
        }
        if (!have) load();  // the first ones, or one episode at a time again
        if (!LOCAL) put_row<BF, P>(tid, Qs, q, lo, hi, !once);
        put_row<BF, P>(tid, Ks, k, lo, hi, !once);
        put_row<BF, P>(tid, Vs, v, lo, hi, !once);
        if (!LOCAL) put_norm<BF, P>(tid, R.rq, q, lo, hi);
        put_norm<BF, P>(tid, R.rk, k, lo, hi);
        if (!once && w == NT - 1) fill_rows<CH>(tid, R, g, A, lo, hi);
        __syncthreads();
        have = once;
        if (once) {  // the next chunk's are on their way while this one computes
          walk(1);
          rows = rows_at(t0 + CH);
          load();
        }
        if (R.starts >> lo & 1) {  // whatever the steps before left
#pragma unroll
          for (int m = 0; m < NT; m++) S[m] = zero;
        }
        score_tiles<BF, P, LD, !LOCAL>(tid, R, Qs, Ks, X.M, X.P, diag, scale);
        __syncthreads();
        if (w == 0) invert_blocks<CH>(tid, diag, X.Tinv);
        if (w == NT - 1 && once) fill_rows<CH>(tid, Rs[cur ^ 1], gn, A, 0, rows);
        f4 Y[NB], O[NB];
        {
          Parts<BF> Sp[NT];
#pragma unroll
          for (int m = 0; m < NT; m++) Sp[m].set(S[m]);
#pragma unroll
          for (int n = 0; n < NB; n++) {
            unit x[NT];
#pragma unroll
            for (int m = 0; m < NT; m++) x[m] = row_unit<LD>(tid, Ks, 16 * n, 16 * m);
            const f4 ks = dot_parts<BF, NT>(x, Sp, zero);
            Y[n] = rows4(tid, R.be, 16 * n) * (widen(col_unit<LD>(tid, Vs, 16 * n, 16 * w)) -
                                          (rows4(tid, R.d0, 16 * n) * rows4(tid, R.rk, 16 * n)) * (ks));
            if constexpr (!LOCAL) {
#pragma unroll
              for (int m = 0; m < NT; m++) x[m] = row_unit<LD>(tid, Qs, 16 * n, 16 * m);
              O[n] = (scale * rows4(tid, R.d0, 16 * n) * rows4(tid, R.rq, 16 * n)) * (dot_parts<BF, NT>(x, Sp, zero));
            }
          }
        }
        mark_odd<CH, NB>(tid, R, Y, lo, hi);
        __syncthreads();
        const int starts = R.starts, inside = starts & ~(1 << lo);
        if (__builtin_amdgcn_readfirstlane(R.odd)) {  // only the rows up to the next episode, or to a row that the ones in front may not see
          const int next = inside ? __ffs(inside) - 1 : CH, stop = LOCAL || next < R.split ? next : R.split;
          if (stop < hi) {
            if (once) walk(-1);
            have = false;
            rows = all;
            hi = __builtin_amdgcn_readfirstlane(stop);
            continue;
          }
        }
        f4 U[NB];
        solve<BF>(tid, X.Tinv, X.M, Y, U);
        if constexpr (!LOCAL) {
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int m = 0; m <= n; m++) {
              const f4 x = mat_col<UD>(tid, X.P, 16 * m, 16 * n);
              O[n] = dot<1>(&x, U + m, O[n]);
            }
          // y rests where V was, until the rows are stored behind the next barrier
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) stf(Vs + (16 * n + 4 * (l >> 4) + i) * LD + 16 * w + (l & 15), O[n][i]);
        }
        Parts<BF> Uw[NB];
#pragma unroll
        for (int n = 0; n < NB; n++) Uw[n].set((rows4(tid, R.dc, 16 * n) * rows4(tid, R.rk, 16 * n)) * (U[n]));
        const float c0 = R.c0;
#pragma unroll
        for (int m = 0; m < NT; m++) {
          unit kt[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) kt[n] = col_unit<LD>(tid, Ks, 16 * n, 16 * m);
          S[m] = dot_parts<BF, NB>(kt, Uw, c0 * S[m]);
        }
        cut |= starts;
        y_at = t0;
        y_lo = lo;
        y_hi = hi;
        lo = hi;
        hi = all;
        if (!once && lo >= all) {  // on to the next chunk's rows
          walk(1);
          rows = rows_at(t0 + CH);
        }
      }
      if (w == NT - 1) {
        g = gn;
        gn = load_gate<T>(bt, h, t0 + 2 * CH, rows_at(t0 + 2 * CH), l);
      }
      cur ^= 1;
    }
    if (!LOCAL) {
      __syncthreads();
      put_y(y_at, y_lo, y_hi);
    }
    const Args e = again<Args>(0);
    if (LOCAL) {
      const long at = seg * e.units + unit_id;
      gout<float> out = (gout<float>)(part ? e.phi : e.psi) + at * own.floats();
#pragma unroll
      for (int m = 0; m < NT; m++)
        if (part && e.parts == 2) put_own_tile_t(tid, out, own, m, w, S[m]);  // for Phi S; the gradient takes Phi^T dS
        else put_own_tile(tid, out, own, m, w, S[m]);
      if (part && tid == 0) e.cut[at] = cut != 0;
    } else if (e.h_out && last == e.T) {
      put_state<NT>(tid, (gout<float>)e.h_out + unit_id * e.K * e.V, e.K, e.V, w, S);
    }
  }
}

__host__ __device__ __forceinline__ long join_blocks(const Args& s) { return (s.units + 7) / 8 * 8 * (up16(s.V) / 16); }
// The segments' start states in order, S <- Phi S + Psi (back: the gradients of their end states in reverse, dS <- Phi^T dS + Xi). An
// episode's start in a segment leaves only what the segment adds. A chain of small fp32 products, so it is spread thin: a block
// per 16 columns of a sequence's head, a wavefront per 16 rows, which exchange their tiles through LDS; Phi's come from memory as
// they are needed, DEEP segments ahead. 32 segments of 2 x 8 heads of 64x64 24 us (54 with all columns in one block and Phi in LDS), 8
// of 8 x 4 heads of 128x128 11 to 13 (25; 27 with a head's columns on different XCDs).
template <int P, bool BACK> __global__ void __launch_bounds__(4 * P) k_delta_join(const Args s, const GradArgs o) {
  constexpr int NT = P / 16, DEEP = P <= 64 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) f4 X[2][NT][64];
  __shared__ int cuts[kMostSegments];
  const int tid = threadIdx.x, l = tid & 63, m = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Own own = {up16(s.K) / 16, up16(s.V) / 16}, sq = {own.tk, own.tk};
  const long n = s.segs - 1, items = join_blocks(s);
  for (long item = blockIdx.x; item < items; item += gridDim.x) {
    // a head's columns share its Phi: on one XCD (every eighth block), in whose L2 it then lies
    const long unit_id = item / 8 / own.tv * 8 + item % 8;
    const int w = (int)(item / 8 % own.tv);
    if (unit_id >= s.units) continue;
    __syncthreads();
    for (int i = tid; i < n; i += 4 * P) cuts[i] = s.cut[(BACK ? n - i : i) * s.units + unit_id];
    f4 S = {0.f, 0.f, 0.f, 0.f}, phi[DEEP][NT], add[DEEP];
    const float* from = BACK ? o.dh : s.h0;
    if (from && m < own.tk)
      get_state<1, false>(tid, (gin<float>)from + unit_id * s.K * s.V + 16 * m * s.V, s.K - 16 * m, s.V, w, &S);
    auto out = [&](long i) {  // the state that is handed to segment i, in the order of the passes
      return (gout<float>)(BACK ? o.dend : s.start) + ((BACK ? n - i : i) * s.units + unit_id) * own.floats();
    };
    put_own_tile(tid, out(0), own, m, w, S);
    auto load = [&](int d, long i) {
      const long at = (BACK ? n - i : i) * s.units + unit_id;  // the segment that is passed
      gin<float> f = (gin<float>)s.phi + at * sq.floats();
      add[d] = own_tile(tid, (gin<float>)(BACK ? o.xi : s.psi) + at * own.floats(), own, m, w);
#pragma unroll
      for (int j = 0; j < NT; j++) phi[d][j] = BACK ? own_tile(tid, f, sq, j, m) : own_tile(tid, f, sq, m, j);
    };
#pragma unroll
    for (int d = 0; d < DEEP; d++) load(d, d < n ? d : n - 1);
    for (long i0 = 0; i0 < n; i0 += DEEP) {
#pragma unroll
      for (int d = 0; d < DEEP; d++) {
        const long i = i0 + d;
        if (i >= n) break;
        X[i & 1][m][l] = S;
        __syncthreads();  // tiles of the segment before last may be overwritten: all have read them in front of this
        S = add[d];
        if (!__builtin_amdgcn_readfirstlane(cuts[i])) {
#pragma unroll
          for (int j = 0; j < NT; j++) {
            if (j >= own.tk) break;
            const f4 x = X[i & 1][j][l];
            S = dot<1>(&phi[d][j], &x, S);
          }
        }
        load(d, i + DEEP < n ? i + DEEP : n - 1);
        put_own_tile(tid, out(i + 1), own, m, w, S);
      }
    }
  }
}

// U and dY of a chunk, transposed: [V][step]. For bf16 in their three parts, cut once by who writes them (16 tiles of a chunk, which
// are read 120 times); of 128 columns in fp32, cut by each reader, since the third parts would not fit a block's LDS.
template <bool BF, int P> struct Cols {
  using T = typename Elem<BF>::type;
  static constexpr int UD = Elem<BF>::CH + 4;
  static constexpr bool PARTS = BF && P <= 64;
  std::conditional_t<PARTS, T, float> hi[P * UD];
  T mid[PARTS ? P * UD : 1], low[PARTS ? P * UD : 1];
  // A tile's values at rows 16 w + l % 16, columns `at` + 4 (l / 16) + 0..3; and units.
  __device__ __forceinline__ void put(int tid, int w, int at, f4 v) {
    const int l = tid & 63, o = (16 * w + (l & 15)) * UD + at + 4 * (l >> 4);
    if constexpr (PARTS) {
      Parts<BF> p;
      p.set(v);
      *reinterpret_cast<s4*>(hi + o) = p.hi;
      *reinterpret_cast<s4*>(mid + o) = p.mid;
      *reinterpret_cast<s4*>(low + o) = p.low;
    } else {
      *reinterpret_cast<f4*>(hi + o) = v;
    }
  }
  __device__ __forceinline__ Parts<BF> col(int tid, int row, int col) const {
    Parts<BF> p;
    if constexpr (PARTS) {
      p.hi = col_unit<UD>(tid, hi, row, col);
      p.mid = col_unit<UD>(tid, mid, row, col);
      p.low = col_unit<UD>(tid, low, row, col);
    } else {
      p.set(col_unit<UD>(tid, hi, row, col));
    }
    return p;
  }
  __device__ __forceinline__ Parts<BF> row(int tid, int row, int col) const {
    Parts<BF> p;
    if constexpr (PARTS) {
      p.hi = row_unit<UD>(tid, hi, row, col);
      p.mid = row_unit<UD>(tid, mid, row, col);
      p.low = row_unit<UD>(tid, low, row, col);
    } else {
      p.set(row_unit<UD>(tid, hi, row, col));
    }
    return p;
  }
  __device__ __forceinline__ f4 values(int tid, int r, int c) const {
    if constexpr (PARTS) return row(tid, r, c).sum();
    else return row_unit<UD>(tid, hi, r, c);
  }
};

// The gradient of one segment of one sequence's head, chunks in reverse. Wavefront w holds dS's columns 16 w .. and, for the
// products that contract over V, the transposed dS's (rows 16 w .. of dS). LOCAL: what the segment adds to dS alone.
template <bool BF, int P> struct BwdLds {
  using T = typename Elem<BF>::type;
  static constexpr int CH = Elem<BF>::CH, LD = P + Elem<BF>::pad, UD = CH + 4, CP = CH + 4, NT = P / 16;
  T Q[CH * LD], K[CH * LD], dO[CH * LD];
  // V rests where U comes: it is read before.
  union {
    T V[CH * LD];
    Cols<BF, P> U;
    float sums[4][NT][CH];  // when U has been read: <q^, dQ^>, <k^, dK^>, the parts of S_0 and of dS_c
  };
  Cols<BF, P> dY;
  Mat<CH * UD> M;   // then F
  Mat<CH * UD> Pm;  // then E
  union {
    Mat<CH * 20> Tinv;
    float W[CH * CP];  // P_ij dO_i U_j - M_ij dY_i U_j
  };
  union {
    float diag[CH * 16];
    struct {
      float ysum[NT][CH], pairs[CH / 16][CH], tot[NT];
    };
  };
  Rows<CH> R[2];
};
template <bool BF, int P> struct BwdLocalLds {
  using T = typename Elem<BF>::type;
  static constexpr int CH = Elem<BF>::CH, LD = P + Elem<BF>::pad, CP = CH + 4, UD = CH + 4;
  T Q[CH * LD], K[CH * LD], dO[CH * LD];
  Mat<CH * UD> M, Pm;
  Mat<CH * 20> Tinv;
  float diag[CH * 16];
  Rows<CH> R[2];
};

__device__ __forceinline__ float row16_sum(float v) {
  v += dpp_mov<0xB1>(v);
  v += dpp_mov<0x4E>(v);
  v += dpp_mov<0x141>(v);
  v += dpp_mov<0x140>(v);
  return v;
}

template <bool BF, int P, bool LOCAL>
__global__ void __launch_bounds__(4 * P, (bwd_waves<BF, P>())) k_delta_bwd(const Args args, const GradArgs gargs) {
  using T = typename Elem<BF>::type;
  using unit = typename Elem<BF>::unit;
  using Lds = std::conditional_t<LOCAL, BwdLocalLds<BF, P>, BwdLds<BF, P>>;
  constexpr int CH = Lds::CH, NB = CH / 16, NT = P / 16, LD = Lds::LD, CP = Lds::CP, UD = CH + 4;
  constexpr int TILES = NB * (NB + 1) / 2;
  static_assert(sizeof(Lds) <= kMaxLdsBytes, "LDS of a block");
  __shared__ __attribute__((aligned(16))) Lds L;
  int tid = threadIdx.x, l = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  for (long item = blockIdx.x;; item += gridDim.x) {
    const Args s = again<Args>(0);
    const GradArgs o = again<GradArgs>(sizeof(Args));
    if (item >= s.units * (LOCAL ? s.segs - 1 : s.segs)) break;
    const unsigned units = (unsigned)s.units, round = (unsigned)item / units;
    const long unit_id = (unsigned)item - round * units, seg = round + (LOCAL ? 1 : 0), bt = (unsigned)unit_id / (unsigned)s.H;
    const int h = (int)(unit_id - bt * s.H), hk = (int)((unsigned)h / (unsigned)(s.H / s.Hk));
    const Own own = {up16(s.K) / 16, up16(s.V) / 16};
    const long c_first = seg * s.seg_chunks, c_all = (s.T + CH - 1) / CH;
    long c = c_first + s.seg_chunks < c_all ? c_first + s.seg_chunks - 1 : c_all - 1;
    gin<T> qp = thread_row<BF, P>(tid, (const T*)s.q + bt * s.q_b + hk * s.q_h, s.q_t, c * CH);
    gin<T> kp = thread_row<BF, P>(tid, (const T*)s.k + bt * s.k_b + hk * s.k_h, s.k_t, c * CH);
    gin<T> vp = thread_row<BF, P>(tid, (const T*)s.v + bt * s.v_b + h * s.v_h, s.v_t, c * CH);
    gin<T> op = thread_row<BF, P>(tid, (const T*)o.dy + bt * o.dy_b + h * o.dy_h, o.dy_t, c * CH);
    const float A = s.A[h], scale = s.scale;
    const long steps = s.T;
    auto rows_at = [&](long ch) { return (int)(ch < c_first ? 0 : steps - ch * CH < CH ? steps - ch * CH : CH); };
    double sumA = 0.0, sumB = 0.0;  // of the lanes that see to the gates
    f4 dS[NT], dSt[LOCAL ? 1 : NT];
    if (!LOCAL && s.segs > 1) {
      gin<float> d = (gin<float>)o.dend + (seg * s.units + unit_id) * own.floats();
#pragma unroll
      for (int m = 0; m < NT; m++) {
        dS[m] = own_tile(tid, d, own, m, w);
        if (m >= own.tk || w >= own.tv) dS[m] = zero;
        if constexpr (!LOCAL) {
          dSt[m] = own_tile_t(tid, d, own, m, w);
          if (m >= own.tv || w >= own.tk) dSt[m] = zero;
        }
      }
    } else if (!LOCAL && o.dh) {
      get_state<NT, false>(tid, (gin<float>)o.dh + unit_id * s.K * s.V, s.K, s.V, w, dS);
      if constexpr (!LOCAL) get_state<NT, true>(tid, (gin<float>)o.dh + unit_id * s.K * s.V, s.K, s.V, w, dSt);
    } else {
#pragma unroll
      for (int m = 0; m < NT; m++) {
        dS[m] = zero;
        if constexpr (!LOCAL) dSt[m] = zero;
      }
    }
    int rows = rows_at(c);
    u4 q, k, v = {0, 0, 0, 0}, d;
    auto load = [&]() {
      const Args a = again<Args>(0);
      q = load_row<BF, P>(tid, qp, rows, a.K);
      k = load_row<BF, P>(tid, kp, rows, a.K);
      if (!LOCAL) v = load_row<BF, P>(tid, vp, rows, a.V);
      d = load_row<BF, P>(tid, op, rows, a.V);
    };
    auto walk = [&](int chunks) {
      const Args a = again<Args>(0);
      const GradArgs b = again<GradArgs>(sizeof(Args));
      qp += chunks * CH * a.q_t;
      kp += chunks * CH * a.k_t;
      vp += chunks * CH * a.v_t;
      op += chunks * CH * b.dy_t;
    };
    bool have = false;  // this chunk's rows are there
    auto next = [&]() {  // the next chunk's rows are on their way while this one computes
      walk(-1);
      rows = rows_at(c - 1);
      load();
      have = true;
    };
    auto keep_at = [&](long ch) {
      const Args a = again<Args>(0);
      return (gin<float>)again<GradArgs>(sizeof(Args)).keep + (ch * a.units + unit_id) * own.floats();
    };
    // the last wavefront sees to the gates, a chunk ahead
    Gate<T> g = {}, gn = g;
    if (w == NT - 1) {
      g = load_gate<T>(bt, h, c * CH, rows, l);
      gn = load_gate<T>(bt, h, (c - 1) * CH, rows_at(c - 1), l);
    }
    __syncthreads();  // the item before has been read
    if (w == NT - 1) fill_rows<CH>(tid, L.R[0], g, A, 0, rows);
    int cur = 0, y_lo = 0, y_hi = 0;
    long y_at = 0;
    auto put_grads = [&](long at, int lo, int hi) {  // a thread stores the 16 bytes that it stages next
      const GradArgs a = again<GradArgs>(sizeof(Args));
      const Args sa = again<Args>(0);
      const int row = tid / (P / Elem<BF>::V), c = tid % (P / Elem<BF>::V) * Elem<BF>::V, from = row * LD + c;
      if (row < lo || row >= hi) return;
      if (a.dv) store_row<BF>((gout<T>)a.dv + bt * a.dv_b + h * a.dv_h + (at + row) * a.dv_t + c, L.dO + from, sa.V - c);
      if (a.dq && !a.qpart) store_row<BF>((gout<T>)a.dq + bt * a.dq_b + h * a.dq_h + (at + row) * a.dq_t + c, L.Q + from, sa.K - c);
      if (a.dk && !a.qpart) store_row<BF>((gout<T>)a.dk + bt * a.dk_b + h * a.dk_h + (at + row) * a.dk_t + c, L.K + from, sa.K - c);
    };
    for (; c >= c_first; c--) {
      Rows<CH>& R = L.R[cur];
      const long t0 = c * CH;
      const int all = rows;  // rows of this chunk
      for (int lo = 0, hi = all, once = 1; hi > 0; once = 0) {
        __syncthreads();  // the rows before have been read
        renew(tid, l);
        if constexpr (!LOCAL) {
          put_grads(y_at, y_lo, y_hi);
          y_hi = 0;
        }
        if (!have) load();  // the first ones, or one episode at a time again
        have = false;
        put_row<BF, P>(tid, L.Q, q, lo, hi, !once);
        put_row<BF, P>(tid, L.K, k, lo, hi, !once);
        if constexpr (!LOCAL) put_row<BF, P>(tid, L.V, v, lo, hi, !once);
        put_row<BF, P>(tid, L.dO, d, lo, hi, !once);
        bool odd = put_norm<BF, P>(tid, R.rq, q, lo, hi);
        odd |= put_norm<BF, P>(tid, R.rk, k, lo, hi);
        odd |= tid / (P / Elem<BF>::V) >= lo && tid / (P / Elem<BF>::V) < hi && !all_near<BF>(d);
        if (!once && w == NT - 1) fill_rows<CH>(tid, R, g, A, lo, hi);
        f4 S0[LOCAL ? 1 : NT];
        if constexpr (!LOCAL) {
#pragma unroll
          for (int m = 0; m < NT; m++) S0[m] = own_tile(tid, keep_at(c), own, m, w);
        }
        __syncthreads();
        const bool fresh = R.starts >> lo & 1;  // S_0 may be anything
        score_tiles<BF, P, LD, true>(tid, R, L.Q, L.K, L.M, L.Pm, L.diag, scale);
        __syncthreads();
        if (w == 0) invert_blocks<CH>(tid, L.diag, L.Tinv);
        if (w == NT - 1 && once) fill_rows<CH>(tid, L.R[cur ^ 1], gn, A, 0, rows_at(c - 1));
        // contractions over the state's rows, HT tiles at a time: the operands of all would not fit the registers
        constexpr int HT = 2;
        f4 Y[NB], dU[NB], sd = zero;
#pragma unroll
        for (int n = 0; n < NB; n++) Y[n] = dU[n] = zero;
#pragma unroll
        for (int m0 = 0; m0 < NT; m0 += HT) {
          Parts<BF> Sp[HT], Dp[HT];
#pragma unroll
          for (int m = 0; m < HT; m++) {
            if constexpr (!LOCAL) {
              if (fresh) S0[m0 + m] = zero;
              sd += S0[m0 + m] * dS[m0 + m];
              Sp[m].set(S0[m0 + m]);
            }
            Dp[m].set(dS[m0 + m]);
          }
#pragma unroll
          for (int n = 0; n < NB; n++) {
            unit x[HT];
#pragma unroll
            for (int m = 0; m < HT; m++) x[m] = row_unit<LD>(tid, L.K, 16 * n, 16 * (m0 + m));
            if constexpr (!LOCAL) Y[n] = dot_parts<BF, HT>(x, Sp, Y[n]);
            dU[n] = dot_parts<BF, HT>(x, Dp, dU[n]);
          }
          if (NT > 4) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < NB; n++) {
          const f4 rk = rows4(tid, R.rk, 16 * n);
          if constexpr (!LOCAL)
            Y[n] = rows4(tid, R.be, 16 * n) * (widen(col_unit<LD>(tid, L.V, 16 * n, 16 * w)) - rows4(tid, R.d0, 16 * n) * rk * Y[n]);
          dU[n] = rows4(tid, R.dc, 16 * n) * rk * dU[n];
        }
        {  // what would pass to other episodes in the products, before it does
          bool any = odd;
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) any |= (!LOCAL && !(fabsf(Y[n][i]) < kFar)) || !(fabsf(dU[n][i]) < kFar);
          if (any) R.odd = 1;
        }
        __syncthreads();
        renew(tid, l);
        const int starts = R.starts, inside = starts & ~(1 << lo);
        if (inside && __builtin_amdgcn_readfirstlane(R.odd)) {
          lo = 31 - __clz(inside);
          continue;
        }
        // U, dU, dY: this wavefront's columns of V
        f4 U[NB], dY[NB];
        unit dOc[NB];
        {
          if constexpr (!LOCAL) solve<BF>(tid, L.Tinv, L.M, Y, U);
#pragma unroll
          for (int m = 0; m < NB; m++) {
            dOc[m] = col_unit<LD>(tid, L.dO, 16 * m, 16 * w);
            const f4 d = widen(dOc[m]);
#pragma unroll
            for (int n = 0; n <= m; n++) {
              const f4 x = mat_row<UD>(tid, L.Pm, 16 * n, 16 * m);
              dU[n] = dot<1>(&x, &d, dU[n]);
            }
          }
          solve_t<BF>(tid, L.Tinv, L.M, dU, dY);
        }
        const int col = 16 * w + (l & 15);
        if constexpr (!LOCAL) {
#pragma unroll
          for (int n = 0; n < NB; n++) {
            L.U.put(tid, w, 16 * n, U[n]);
            L.dY.put(tid, w, 16 * n, dY[n]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float sum = row16_sum(dY[n][i] * U[n][i]);
              if ((l & 15) == 0) L.ysum[w][16 * n + 4 * (l >> 4) + i] = sum;
            }
          }
        }
        if (LOCAL && once) next();
        const float c0 = R.c0;
        float tot = c0 == 0.f ? 0.f : c0 * (sd[0] + sd[1] + sd[2] + sd[3]);
        // dS of the chunk's start; the transposed one below, when its old values have been used
        {
          Parts<BF> x[NB], y[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) {
            x[n].set((scale * rows4(tid, R.d0, 16 * n) * rows4(tid, R.rq, 16 * n)) * (widen(dOc[n])));
            y[n].set((-rows4(tid, R.d0, 16 * n) * rows4(tid, R.rk, 16 * n) * rows4(tid, R.be, 16 * n)) * (dY[n]));
          }
#pragma unroll
          for (int m = 0; m < NT; m++) {
            unit a[NB];
#pragma unroll
            for (int n = 0; n < NB; n++) a[n] = col_unit<LD>(tid, L.Q, 16 * n, 16 * m);
            dS[m] = dot_parts<BF, NB>(a, x, c0 * dS[m]);
#pragma unroll
            for (int n = 0; n < NB; n++) a[n] = col_unit<LD>(tid, L.K, 16 * n, 16 * m);
            dS[m] = dot_parts<BF, NB>(a, y, dS[m]);
            if (NT > 4) __builtin_amdgcn_sched_barrier(0);  // or the operands of all tiles are loaded at once, and do not fit
          }
        }
        if constexpr (!LOCAL) {
#pragma unroll
          for (int m = 0; m < NT; m++) S0[m] = own_tile_t(tid, keep_at(c), own, m, w);
          __syncthreads();
        renew(tid, l);
          for (int tile = w; tile < TILES; tile += NT) {
            const int bi = tile == 0 ? 0 : 1, bj = tile == 2 ? 1 : 0;  // (0,0) (1,0) (1,1)
            f4 e = zero, f = zero;
#pragma unroll
            for (int m0 = 0; m0 < NT; m0 += HT) {
              Parts<BF> y[HT], x[HT];
              unit z[HT];
#pragma unroll
              for (int m = 0; m < HT; m++) {
                y[m] = L.U.col(tid, 16 * (m0 + m), 16 * bj);
                z[m] = row_unit<LD>(tid, L.dO, 16 * bi, 16 * (m0 + m));
                x[m] = L.dY.col(tid, 16 * (m0 + m), 16 * bi);
              }
              e = dot_parts<BF, HT>(z, y, e);
              f = dot_parts<BF, HT>(x, y, f);
              if (NT > 4) __builtin_amdgcn_sched_barrier(0);
            }
            const int j = 16 * bj + (l & 15);
            const double Gj = R.G[j];
            const int segj = R.seg[j];
            const f4 pv = mat_row<UD>(tid, L.Pm, 16 * bj, 16 * bi), mv = mat_row<UD>(tid, L.M, 16 * bj, 16 * bi);
            const f4 be = rows4(tid, R.be, 16 * bi);
#pragma unroll
            for (int i4 = 0; i4 < 4; i4++) {
              const int i = 16 * bi + 4 * (l >> 4) + i4;
              const bool on = segj == R.seg[i] && j <= i;
              const float dec = ex2((float)(R.G[i] - Gj));
              L.W[i * CP + j] = on && j < i ? pv[i4] * e[i4] - mv[i4] * f[i4] : 0.f;
              e[i4] = on ? dec * scale * e[i4] : 0.f;
              f[i4] = on && j < i ? -dec * be[i4] * f[i4] : 0.f;
            }
            put_mat<UD>(tid, L.Pm, 16 * bj, 16 * bi, e);
            put_mat<UD>(tid, L.M, 16 * bj, 16 * bi, f);
          }
          renew(tid, l);
          // products over V for this wavefront's columns of K: dO S_0^T, dY S_0^T, U dS^T
          f4 X1[NB], X2[NB], X3[NB];
#pragma unroll
          for (int n = 0; n < NB; n++) X1[n] = X2[n] = X3[n] = zero;
#pragma unroll
          for (int m0 = 0; m0 < NT; m0 += HT) {
            Parts<BF> St[HT], Dt[HT];
#pragma unroll
            for (int m = 0; m < HT; m++) {
              St[m].set(fresh ? zero : S0[m0 + m]);
              Dt[m].set(dSt[m0 + m]);
            }
#pragma unroll
            for (int n = 0; n < NB; n++) {
              unit x[HT];
#pragma unroll
              for (int m = 0; m < HT; m++) x[m] = row_unit<LD>(tid, L.dO, 16 * n, 16 * (m0 + m));
              X1[n] = dot_parts<BF, HT>(x, St, X1[n]);
              Parts<BF> y[HT];
#pragma unroll
              for (int m = 0; m < HT; m++) y[m] = L.dY.col(tid, 16 * (m0 + m), 16 * n);
              X2[n] = dot_parts<BF, HT>(y, St, X2[n]);
#pragma unroll
              for (int m = 0; m < HT; m++) y[m] = L.U.col(tid, 16 * (m0 + m), 16 * n);
              X3[n] = dot_parts<BF, HT>(y, Dt, X3[n]);
              if (NT > 4) __builtin_amdgcn_sched_barrier(0);
            }
          }
#pragma unroll
          for (int n = 0; n < NB; n++) {
            const f4 d0 = rows4(tid, R.d0, 16 * n);
            X1[n] = scale * d0 * X1[n];
            X2[n] = -d0 * rows4(tid, R.be, 16 * n) * X2[n];
            X3[n] = rows4(tid, R.dc, 16 * n) * X3[n];
          }
        renew(tid, l);
          unit Kc[NB], Qc[NB];  // this wavefront's columns of K and Q
#pragma unroll
          for (int n = 0; n < NB; n++) {
            Kc[n] = col_unit<LD>(tid, L.K, 16 * n, 16 * w);
            Qc[n] = col_unit<LD>(tid, L.Q, 16 * n, 16 * w);
          }
          {
            Parts<BF> x[NB], y[NB];
#pragma unroll
            for (int n = 0; n < NB; n++) {
              x[n].set((scale * rows4(tid, R.d0, 16 * n) * rows4(tid, R.rq, 16 * n)) * (widen(Qc[n])));
              y[n].set((-rows4(tid, R.d0, 16 * n) * rows4(tid, R.rk, 16 * n) * rows4(tid, R.be, 16 * n)) * (widen(Kc[n])));
            }
#pragma unroll
            for (int m = 0; m < NT; m++) {
              unit a[NB];
#pragma unroll
              for (int n = 0; n < NB; n++) a[n] = col_unit<LD>(tid, L.dO, 16 * n, 16 * m);
              dSt[m] = dot_parts<BF, NB>(a, x, c0 * dSt[m]);
              Parts<BF> b[NB];
#pragma unroll
              for (int n = 0; n < NB; n++) b[n] = L.dY.row(tid, 16 * m, 16 * n);
              dSt[m] = dot_parts<BF, NB>(b, y, dSt[m]);
              if (NT > 4) __builtin_amdgcn_sched_barrier(0);
            }
          }
          __syncthreads();
        renew(tid, l);
          if (once) next();
          // E K^, F K^ (rows as i), F^T K^, E^T Q^ (rows as j): E and F rest where P and M were
          f4 dQ[NB], dK[NB];
          {
            f4 qn[NB], kn[NB];
#pragma unroll
            for (int n = 0; n < NB; n++) {
              qn[n] = widen(Qc[n]) * rows4(tid, R.rq, 16 * n);
              kn[n] = widen(Kc[n]) * rows4(tid, R.rk, 16 * n);
            }
#pragma unroll
            for (int n = 0; n < NB; n++) {
              const f4 from0 = qn[n] * X1[n] + kn[n] * X2[n], fromc = kn[n] * X3[n];
              dQ[n] = X1[n];
              dK[n] = X2[n] + X3[n];
#pragma unroll
              for (int m = 0; m < NB; m++) {  // F and F^T take K^ both
                f4 f = zero;
                if (m <= n) {
                  const f4 e = mat_col<UD>(tid, L.Pm, 16 * m, 16 * n);
                  dQ[n] = dot<1>(&e, kn + m, dQ[n]);
                  f = mat_col<UD>(tid, L.M, 16 * m, 16 * n);
                }
                if (m >= n) {
                  const f4 e = mat_row<UD>(tid, L.Pm, 16 * n, 16 * m);
                  dK[n] = dot<1>(&e, qn + m, dK[n]);
                  f += mat_row<UD>(tid, L.M, 16 * n, 16 * m);
                }
                dK[n] = dot<1>(&f, kn + m, dK[n]);
              }
              const f4 sq = qn[n] * dQ[n], sk = kn[n] * dK[n];
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const float x[4] = {row16_sum(sq[i]), row16_sum(sk[i]), row16_sum(from0[i]), row16_sum(fromc[i])};
                if ((l & 15) == 0) {
#pragma unroll
                  for (int j = 0; j < 4; j++) L.sums[j][w][16 * n + 4 * (l >> 4) + i] = x[j];
                }
              }
            }
          }
          // sums over the pairs j < t <= i, rows t: a triangle of ones times W, then along the row
          for (int tile = w; tile < TILES; tile += NT) {
            const int bt_ = tile == 0 ? 0 : 1, bj = tile == 2 ? 1 : 0, t = 16 * bt_ + (l & 15);
            f4 acc = zero;
            for (int m = bt_; m < NB; m++) {
              f4 ones;
#pragma unroll
              for (int i = 0; i < 4; i++) ones[i] = 16 * m + 4 * (l >> 4) + i >= t ? 1.f : 0.f;
              const f4 x = col_unit<CP>(tid, L.W, 16 * m, 16 * bj);
              acc = dot<1>(&ones, &x, acc);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int row = 16 * bt_ + 4 * (l >> 4) + i;
              const float sum = row16_sum(16 * bj + (l & 15) < row ? acc[i] : 0.f);
              if ((l & 15) == 0) L.pairs[bj][row] = sum;
            }
          }
          tot = group_sum<64>(tot);
          if (l == 0) L.tot[w] = tot;
          __syncthreads();
        renew(tid, l);
          // through the norms; dq, dk and dv rest where Q, K and dO were, until the rows are stored behind the next barrier
          const GradArgs a = again<GradArgs>(sizeof(Args));
          const Args sa = again<Args>(0);
#pragma unroll
          for (int n = 0; n < NB; n++) {
            const f4 rq = rows4(tid, R.rq, 16 * n), rk = rows4(tid, R.rk, 16 * n), be = rows4(tid, R.be, 16 * n);
            f4 sq = zero, sk = zero;
#pragma unroll
            for (int m = 0; m < NT; m++) {
              sq += rows4(tid, L.sums[0][m], 16 * n);
              sk += rows4(tid, L.sums[1][m], 16 * n);
            }
            const f4 dq = rq * (dQ[n] - widen(Qc[n]) * rq * sq), dk = rk * (dK[n] - widen(Kc[n]) * rk * sk);
            const f4 dv = be * L.dY.values(tid, 16 * w, 16 * n);
            if (a.qpart) {
              const unsigned step = (unsigned)(sa.H * sa.K);  // elements of a sequence's step
              const long to = (((t0 + 16 * n + 4 * (l >> 4)) * sa.B + bt) * sa.H + h) * sa.K + col;
#pragma unroll 1
              for (int i = 0; i < 4; i++) {
                const int row = 16 * n + 4 * (l >> 4) + i;
                if (row >= lo && row < hi && col < sa.K) {
                  const float x = i == 0 ? dq[0] : i == 1 ? dq[1] : i == 2 ? dq[2] : dq[3], z = i == 0 ? dk[0] : i == 1 ? dk[1] : i == 2 ? dk[2] : dk[3];
                  ((gout<float>)a.qpart)[to + (long)i * sa.B * step] = x;
                  ((gout<float>)a.kpart)[to + (long)i * sa.B * step] = z;
                }
              }
            }
            const int at = (16 * n + 4 * (l >> 4)) * LD + col;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              stf(L.dO + at + i * LD, dv[i]);
              stf(L.Q + at + i * LD, dq[i]);
              stf(L.K + at + i * LD, dk[i]);
            }
          }
          y_at = t0;
          y_lo = lo;
          y_hi = hi;
          if (w == NT - 1) {  // the gates
            float from0 = 0.f, fromc = 0.f, dbr = 0.f, sum = 0.f;
            const int i = l < CH ? l : CH - 1;
#pragma unroll
            for (int m = 0; m < NT; m++) {
              from0 += L.sums[2][m][i];
              fromc += L.sums[3][m][i];
              dbr += L.ysum[m][i];
              sum += L.tot[m];
            }
            from0 += dpp_mov<0x101>(from0);  // of the rows from t on: sums along the rows of 16 lanes
            from0 += dpp_mov<0x102>(from0);
            from0 += dpp_mov<0x104>(from0);
            from0 += dpp_mov<0x108>(from0);
            fromc += dpp_mov<0x111>(fromc);  // of the rows up to t
            fromc += dpp_mov<0x112>(fromc);
            fromc += dpp_mov<0x114>(fromc);
            fromc += dpp_mov<0x118>(fromc);
            const float low = lane_f32(fromc, 15);
            fromc = dpp_mov<0x111>(fromc);  // and before t
            if constexpr (NB == 2) {
              const float high = lane_f32(from0, 16);
              if (l < 16) from0 += high;
              else fromc += low;
            }
            float dg = L.pairs[0][i] + from0 + fromc + sum;
            if (NB == 2 && i >= 16) dg += L.pairs[NB - 1][i];
            if (l >= lo && l < hi) {
              const float be = R.be[l], arg = R.arg[l];
              const float da = dg * A * sigma(arg);
              if (a.da) stf((gout<T>)a.da + (t0 + l) * a.da_t + bt * a.da_b + h, da);
              if (a.db) stf((gout<T>)a.db + (t0 + l) * a.db_t + bt * a.db_b + h, dbr * (1.f - be));
              sumA += (double)dg * (double)R.sp[l];
              sumB += (double)da;
            }
          }
        }
        if (starts >> lo & 1) {  // nothing passes to the steps before, whatever these hold
#pragma unroll
          for (int m = 0; m < NT; m++) {
            dS[m] = zero;
            if constexpr (!LOCAL) dSt[m] = zero;
          }
        }
        hi = lo;
        lo = 0;
        if (!once && hi <= 0) {  // on to the next chunk's rows
          walk(-1);
          rows = rows_at(c - 1);
        }
      }
      if (w == NT - 1) {
        g = gn;
        gn = load_gate<T>(bt, h, (c - 2) * CH, rows_at(c - 2), l);
      }
      cur ^= 1;
    }
    if constexpr (!LOCAL) {
      __syncthreads();
      put_grads(y_at, y_lo, y_hi);
    }
    const Args e = again<Args>(0);
    const GradArgs eo = again<GradArgs>(sizeof(Args));
    if (LOCAL) {
#pragma unroll
      for (int m = 0; m < NT; m++) put_own_tile(tid, (gout<float>)eo.xi + (seg * e.units + unit_id) * own.floats(), own, m, w, dS[m]);
    } else {
      if (eo.dh0 && seg == 0) put_state<NT>(tid, (gout<float>)eo.dh0 + unit_id * e.K * e.V, e.K, e.V, w, dS);
      if (w == NT - 1 && eo.gpart) {
#pragma unroll
        for (int d2 = 1; d2 < CH; d2 *= 2) {
          sumA += __shfl_xor(sumA, d2);
          sumB += __shfl_xor(sumB, d2);
        }
        if (l == 0) {
          const long n = e.segs * e.B, at = seg * e.B + bt;
          eo.gpart[(long)h * n + at] = (float)sumA;
          eo.gpart[((long)e.H + h) * n + at] = (float)sumB;
        }
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
// l the columns V (l % LPR) .. of the rows l / LPR, + 64 / LPR, ..., all in registers between the two passes over them. 4096 x 8 heads of
// 64x64 bf16 195 us, 5.6 TB/s; 1024 x 8 of 128x128 237 us, 4.5 TB/s (one wavefront a SIMD); of 128x63, whose rows no 16-byte access
// fits, 296 us, 1.8 TB/s (a column a lane, 57 registers spilled).
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
    const float rk = kk == INFINITY ? NAN : __builtin_amdgcn_rsqf(kk + kEps), rq = qq == INFINITY ? NAN : __builtin_amdgcn_rsqf(qq + kEps);
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
  PH_REQUIRE(p.T <= (1u << 30) && p.B <= (1u << 24) && p.B * p.H < (1ull << 30), "%s: T = %zu, B = %zu, H = %zu out of range",
             who, p.T, p.B, p.H);
  PH_REQUIRE(p.scale == p.scale, "%s: scale is not a number", who);
  if (p.T == 0 || p.B == 0) return PH_OK;
  PH_REQUIRE(p.q && p.k && p.v && p.a && p.b && p.A, "%s: q, k, v, a, b or A missing", who);
  return PH_OK;
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
  return a;
}

int padded(const Args& a) {
  const int d = a.K > a.V ? a.K : a.V;
  return d <= 32 ? 32 : d <= 64 ? 64 : 128;
}
unsigned blocks_of(long n) { return (unsigned)(n < kMaxBlocks ? n : kMaxBlocks); }

// Calls f with the padded size as a constant.
template <typename F> void by_size(const Args& a, F f) {
  switch (padded(a)) {
    case 32: f(std::integral_constant<int, 32>()); break;
    case 64: f(std::integral_constant<int, 64>()); break;
    default: f(std::integral_constant<int, 128>());
  }
}

template <bool BF> int fwd_t(const Args& a, hipStream_t st) {
  by_size(a, [&](auto p) {
    constexpr int P = decltype(p)::value;
    if (a.segs > 1) {
      k_delta_fwd<BF, P, true><<<blocks_of(a.units * (a.segs - 1) * a.parts), 4 * P, 0, st>>>(a);
      k_delta_join<P, false><<<blocks_of(join_blocks(a)), 4 * P, 0, st>>>(a, GradArgs{});
    }
    k_delta_fwd<BF, P, false><<<blocks_of(a.units * a.segs), 4 * P, 0, st>>>(a);
  });
  PH_LAUNCH_CHECK();
  return PH_OK;
}

template <bool BF> int bwd_t(const Args& a, const GradArgs& o, float* dA, float* dbias, hipStream_t st) {
  using T = typename Elem<BF>::type;
  by_size(a, [&](auto p) {
    constexpr int P = decltype(p)::value;
    if (a.segs > 1) {
      k_delta_fwd<BF, P, true><<<blocks_of(a.units * (a.segs - 1)), 4 * P, 0, st>>>(a);
      k_delta_bwd<BF, P, true><<<blocks_of(a.units * (a.segs - 1)), 4 * P, 0, st>>>(a, o);
      k_delta_join<P, true><<<blocks_of(join_blocks(a)), 4 * P, 0, st>>>(a, o);
    }
    k_delta_bwd<BF, P, false><<<blocks_of(a.units * a.segs), 4 * P, 0, st>>>(a, o);
  });
  PH_LAUNCH_CHECK();
  if (o.gpart) {
    k_delta_fold_gates<<<2 * a.H, 256, 0, st>>>(o.gpart, a.segs * a.B, a.H, dA, dbias);
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

// Segments of time, and where their states are: `states` buffers of [segs][units] states, Phi and the cuts.
void set_segments(Args& a, bool grad, int dtype) {
  const long c = dtype == PH_BF16 ? Elem<true>::CH : Elem<false>::CH, chunks = (a.T + c - 1) / c;
  a.segs = (int)delta_segments(chunks, a.units, padded(a));
  a.seg_chunks = (chunks + a.segs - 1) / a.segs;
  a.segs = (int)((chunks + a.seg_chunks - 1) / a.seg_chunks);
  a.local_from = grad ? 1 : 0;
  a.parts = grad ? 1 : 2;
}
long state_floats(const Args& a) { return a.segs > 1 ? a.segs * a.units * up16(a.K) * up16(a.V) : 0; }
long phi_floats(const Args& a) { return a.segs > 1 ? a.segs * a.units * up16(a.K) * up16(a.K) : 0; }

long chunk_steps(int dtype) { return dtype == PH_BF16 ? Elem<true>::CH : Elem<false>::CH; }

// The memory of a call's arrays: blocks read inputs while others write, so no output may share an element with an input.
Span rows_of(const ph_delta_args& p, const void* at, long t, long b, long h, size_t heads, size_t width) {
  const long e = p.dtype == PH_BF16 ? 2 : 4;
  return {at, (long)width * e, {(long)p.T, (long)p.B, (long)heads}, {t * e, b * e, h * e}};
}
Span floats(const void* at, size_t n) { return flat(at, (long)n * 4); }
Span state_of(const ph_delta_args& p, const void* at) { return floats(at, p.B * p.H * p.K * p.V); }
struct Spans {
  Span s[16];
  int n = 0;
  void add(const Span& x) { s[n++] = x; }
  bool meet(const Span& x) const {
    for (int i = 0; i < n; i++)
      if (ph::meet(s[i], x)) return true;
    return false;
  }
};
Spans inputs_of(const ph_delta_args& p, bool seq) {
  Spans in;
  in.add(rows_of(p, p.q, p.q_t, p.q_b, p.q_h, p.Hk, p.K));
  in.add(rows_of(p, p.k, p.k_t, p.k_b, p.k_h, p.Hk, p.K));
  in.add(rows_of(p, p.v, p.v_t, p.v_b, p.v_h, p.H, p.V));
  in.add(rows_of(p, p.a, p.a_t, p.a_b, 0, 1, p.H));
  in.add(rows_of(p, p.b, p.b_t, p.b_b, 0, 1, p.H));
  in.add(floats(p.A, p.H));
  in.add(floats(p.dt_bias, p.H));
  in.add(floats(p.first, p.B));
  if (seq) in.add(floats(p.done, p.T * p.B));
  return in;
}

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" size_t ph_delta_keep_floats(const ph_delta_args* p) {
  if (!p) return 0;
  const size_t c = (size_t)chunk_steps(p->dtype);
  return (p->T + c - 1) / c * p->B * p->H * up16((int)p->K) * up16((int)p->V);
}

extern "C" int ph_delta_scan(const ph_delta_args* p, void* y, long y_t, long y_b, long y_h, float* h_out, float* keep,
                             void* stream) {
  PH_REQUIRE(p, "delta_scan: arguments missing");
  PH_TRY(check(*p, "delta_scan"));
  if (p->B == 0) return PH_OK;
  PH_REQUIRE(p->T >= 1, "delta_scan: no steps");
  PH_REQUIRE(y, "delta_scan: y missing");
  const Span ys = rows_of(*p, y, y_t, y_b, y_h, p->H, p->V), out = state_of(*p, h_out), kept = floats(keep, ph_delta_keep_floats(p));
  Spans in = inputs_of(*p, true);
  PH_REQUIRE(!in.meet(ys) && !meet(state_of(*p, p->h0), ys), "delta_scan: y may not be an input or share elements with one");
  PH_REQUIRE(!folds(ys), "delta_scan: y holds elements twice");
  PH_REQUIRE(!in.meet(out) && !in.meet(kept) && (h_out == p->h0 || !meet(state_of(*p, p->h0), out)) && !meet(state_of(*p, p->h0), kept) &&
                 !meet(ys, out) && !meet(ys, kept) && !meet(out, kept),
             "delta_scan: h_out or the kept states share elements with an input or another output");
  Args a = args_of(*p);
  a.y = y; a.y_t = y_t; a.y_b = y_b; a.y_h = y_h; a.h_out = h_out; a.keep = keep;
  set_segments(a, false, p->dtype);
  if (a.segs > 1) {
    const long ns = state_floats(a), nf = phi_floats(a);
    float* ws = (float*)scratch(kSlotDelta, (size_t)(2 * ns + nf + a.segs * a.units) * 4);
    if (!ws) return PH_ERR_NOMEM;
    a.start = ws;
    a.psi = ws + ns;
    a.phi = ws + 2 * ns;
    a.cut = (int*)(ws + 2 * ns + nf);
  }
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
  Spans in = inputs_of(*p, true);
  in.add(rows_of(*p, dy, dy_t, dy_b, dy_h, p->H, p->V));
  in.add(floats(keep, ph_delta_keep_floats(p)));
  const Span outs[] = {rows_of(*p, g->dq, g->dq_t, g->dq_b, g->dq_h, p->Hk, p->K), rows_of(*p, g->dk, g->dk_t, g->dk_b, g->dk_h, p->Hk, p->K),
                       rows_of(*p, g->dv, g->dv_t, g->dv_b, g->dv_h, p->H, p->V), rows_of(*p, g->da, g->da_t, g->da_b, 0, 1, p->H),
                       rows_of(*p, g->db, g->db_t, g->db_b, 0, 1, p->H), state_of(*p, g->dh0)};
  for (int i = 0; i < 6; i++) {
    PH_REQUIRE(!in.meet(outs[i]) && ((i == 5 && g->dh0 == dh) || !meet(state_of(*p, dh), outs[i])),
               "delta_scan_grad: a gradient may not be an input or share elements with one");
    for (int j = 0; j < i; j++) PH_REQUIRE(!meet(outs[i], outs[j]), "delta_scan_grad: two gradients are the same or share elements");
  }
  for (const Span& out : outs) PH_REQUIRE(!folds(out), "delta_scan_grad: a gradient holds elements twice");
  Args a = args_of(*p);
  GradArgs o{};
  o.dy = dy; o.dy_t = dy_t; o.dy_b = dy_b; o.dy_h = dy_h; o.keep = keep; o.dh = dh;
  o.dq = g->dq; o.dq_t = g->dq_t; o.dq_b = g->dq_b; o.dq_h = g->dq_h;
  o.dk = g->dk; o.dk_t = g->dk_t; o.dk_b = g->dk_b; o.dk_h = g->dk_h;
  o.dv = g->dv; o.dv_t = g->dv_t; o.dv_b = g->dv_b; o.dv_h = g->dv_h;
  o.da = g->da; o.da_t = g->da_t; o.da_b = g->da_b;
  o.db = g->db; o.db_t = g->db_t; o.db_b = g->db_b;
  o.dh0 = g->dh0;
  const bool shared = p->Hk != p->H && (g->dq || g->dk), gates = g->dA || g->ddt_bias;
  set_segments(a, true, p->dtype);
  const size_t nq = shared ? p->T * p->B * p->H * p->K : 0, ng = gates ? 2 * p->H * p->B * a.segs : 0;
  const size_t ns = state_floats(a), nf = phi_floats(a), nc = a.segs > 1 ? a.segs * a.units : 0;
  if (nq + ng + ns) {
    float* ws = (float*)scratch(kSlotDelta, (2 * ns + nf + 2 * nq + ng + nc) * 4);
    if (!ws) return PH_ERR_NOMEM;
    o.dend = ws;
    o.xi = ws + ns;
    a.phi = ws + 2 * ns;
    ws += 2 * ns + nf;
    a.cut = (int*)(ws + 2 * nq + ng);
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
  const Span ys = rows_of(*p, y, 0, y_b, y_h, p->H, p->V), state = state_of(*p, h);
  Spans in = inputs_of(*p, false);
  PH_REQUIRE(!in.meet(ys), "delta_step: y may not be an input or share elements with one");
  PH_REQUIRE(!folds(ys), "delta_step: y holds elements twice");
  PH_REQUIRE(!in.meet(state) && !meet(ys, state), "delta_step: the state shares elements with y or an input");
  Args a = args_of(*p);
  a.y = y; a.y_b = y_b; a.y_h = y_h;
  return p->dtype == PH_BF16 ? step_t<uint16_t>(a, h, as_stream(stream)) : step_t<float>(a, h, as_stream(stream));
}
