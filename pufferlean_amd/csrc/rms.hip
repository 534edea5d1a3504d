// RMS normalisation fused with the residual sum in front of it or the gate behind it, and its gradient.
//
//   r = x + scale add,   n = r rstd,  rstd = 1 / sqrt(avg r^2 + eps),   out = n w silu(z)
//
// With g = dout silu(z): dz = dout n w silu'(z), dn = g w, dr = rstd (dn - n avg(dn n)) + dres, dx = dr, dadd = scale dr,
// and the columns' dw = sum g n, dscale = sum dr add. r is not read back but formed again from x and add, in
// fp32: the stored res has been rounded.
//
// Bound by memory: each array is read or written once. A row lives in the registers of LPR lanes (8..64 of a wavefront, or
// the block's 256), one 16-byte access a lane and array; the lanes walk over many rows with their columns of w, scale and the
// columns' sums in registers, and one partial row per block is added by a second, small launch in a fixed order.
//
// Measured, bf16: 262144 rows of 512 with the residual sum 198 us forward (5.4 TB/s) and 289 us back (5.6 TB/s); 131072 x 8 groups
// of 64 with the gate 77 and 131 us (5.2 and 5.1 TB/s); a copy of 2 GiB reaches 5.2 TB/s here. fp32: the same rows 397 and 398 us, 145 and
// 254 us.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "rows.hpp"
#include "spans.hpp"

namespace ph {
namespace {

constexpr int kThreads = 256;

template <typename T> struct RmsArgs {
  const T *x, *add, *z, *dout, *dres;
  T *out, *res, *dx, *dadd, *dz;
  long ldx, ldadd, ldz, lddout, lddres, ldout, ldres, lddx, lddadd, lddz;
  long rows;  // M G
  int C, G, shift;  // columns of a group; log2 G, or -1
  const float *w, *scale;
  float eps;
  float* rstd;
  const float* crstd;
  float *dw, *dscale, *part, *s2;
};

__device__ __forceinline__ float sig(float v) { return 1.f / (1.f + __expf(-v)); }

// Row of a matrix and column offset of a group's row.
struct At {
  long m;
  int col;
  template <typename A> __device__ __forceinline__ At(const A& a, long row) {
    if (a.G == 1) {
      m = row;
      col = 0;
    } else {
      const unsigned r = (unsigned)row, q = a.shift >= 0 ? r >> a.shift : r / (unsigned)a.G;
      m = q;
      col = (int)(r - q * (unsigned)a.G) * a.C;
    }
  }
};

// Sum over the LPR lanes of a row, in all of them. A block's rows take the sum through one of two LDS buffers in turn, so one
// barrier a row suffices: a buffer is written again only behind the next row's.
template <int LPR> __device__ __forceinline__ float row_sum(float v, float (*sh)[4], int& turn) {
  if constexpr (LPR <= 64) {
    return group_sum<LPR>(v);
  } else {
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) sh[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    v = (sh[turn][0] + sh[turn][1]) + (sh[turn][2] + sh[turn][3]);
    turn ^= 1;
    return v;
  }
}

template <typename T, int V, bool AL, int NCH, int LPR, bool ADD, bool GATE>
__global__ void __launch_bounds__(kThreads) k_rms_fwd(const RmsArgs<T> a) {
  constexpr int E = NCH * V, GPB = kThreads / LPR;
  __shared__ float sh[2][4];
  int turn = 0;
  const int lr = threadIdx.x % LPR;
  float wv[E], sv[ADD ? E : 1];
#pragma unroll
  for (int q = 0; q < NCH; q++) {
    const Cols<V> k((q * LPR + lr) * V, a.C);
    get_weights<V>(k, a.w, 1.f, wv + q * V);
    if constexpr (ADD) get_weights<V>(k, a.scale, 1.f, sv + q * V);
  }
  const float inv = 1.f / (float)a.C;
  for (long row = (long)blockIdx.x * GPB + threadIdx.x / LPR; row < a.rows; row += (long)gridDim.x * GPB) {
    const At at(a, row);
    float v[E], z[GATE ? E : 1];
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      const Cols<V> k((q * LPR + lr) * V, a.C);
      get_cols<V, AL>(k, a.x + at.m * a.ldx + at.col, v + q * V);
      if constexpr (GATE) get_cols<V, AL>(k, a.z + at.m * a.ldz + at.col, z + q * V);
      if constexpr (ADD) {
        float d[V];
        get_cols<V, AL>(k, a.add + at.m * a.ldadd + at.col, d);
#pragma unroll
        for (int i = 0; i < V; i++) v[q * V + i] = fmaf(sv[q * V + i], d[i], v[q * V + i]);
        if (a.res) put_cols<V, AL>(k, a.res + at.m * a.ldres + at.col, v + q * V);
      }
    }
#pragma unroll
    for (int i = 0; i < E; i++) s = fmaf(v[i], v[i], s);
    const float r = 1.f / sqrtf(row_sum<LPR>(s, sh, turn) * inv + a.eps);
    if (lr == 0 && a.rstd) a.rstd[row] = r;
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; i++) {
        o[i] = v[q * V + i] * r * wv[q * V + i];
        if constexpr (GATE) o[i] *= z[q * V + i] * sig(z[q * V + i]);
      }
      put_cols<V, AL>(Cols<V>((q * LPR + lr) * V, a.C), a.out + at.m * a.ldout + at.col, o);
    }
  }
}

template <typename T, int V, bool AL, int NCH, int LPR, bool ADD, bool GATE>
__global__ void __launch_bounds__(kThreads) k_rms_bwd(const RmsArgs<T> a) {
  constexpr int E = NCH * V, GPB = kThreads / LPR;
  __shared__ float sh[2][4];
  int turn = 0;
  const int lr = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  float wv[E], sv[ADD ? E : 1], aw[E], as[ADD ? E : 1];
#pragma unroll
  for (int q = 0; q < NCH; q++) {
    const Cols<V> k((q * LPR + lr) * V, a.C);
    get_weights<V>(k, a.w, 1.f, wv + q * V);
    if constexpr (ADD) get_weights<V>(k, a.scale, 1.f, sv + q * V);
  }
#pragma unroll
  for (int i = 0; i < E; i++) aw[i] = 0.f;
#pragma unroll
  for (int i = 0; i < (ADD ? E : 1); i++) as[i] = 0.f;
  const float inv = 1.f / (float)a.C;
  for (long row = (long)blockIdx.x * GPB + grp; row < a.rows; row += (long)gridDim.x * GPB) {
    const At at(a, row);
    float n[E], g[E], d[ADD ? E : 1], z[GATE ? E : 1], dr[E];
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      const Cols<V> k((q * LPR + lr) * V, a.C);
      get_cols<V, AL>(k, a.x + at.m * a.ldx + at.col, n + q * V);
      get_cols<V, AL>(k, a.dout + at.m * a.lddout + at.col, g + q * V);
      if constexpr (ADD) get_cols<V, AL>(k, a.add + at.m * a.ldadd + at.col, d + q * V);
      if constexpr (GATE) get_cols<V, AL>(k, a.z + at.m * a.ldz + at.col, z + q * V);
      if (a.dres) {
        get_cols<V, AL>(k, a.dres + at.m * a.lddres + at.col, dr + q * V);
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) dr[q * V + i] = 0.f;
      }
    }
    const float r = a.crstd[row];
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) {
      if constexpr (ADD) n[i] = fmaf(sv[i], d[i], n[i]);
      n[i] *= r;
      if constexpr (GATE) {
        const float p = sig(z[i]), o = n[i] * wv[i] * g[i];
        g[i] *= z[i] * p;
        z[i] = o * p * fmaf(z[i], 1.f - p, 1.f);
      }
      aw[i] = fmaf(g[i], n[i], aw[i]);
      g[i] *= wv[i];
      s2 = fmaf(g[i], n[i], s2);
    }
    s2 = row_sum<LPR>(s2, sh, turn) * inv;
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      const Cols<V> k((q * LPR + lr) * V, a.C);
      float o[V];
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int e = q * V + i;
        o[i] = fmaf(r, g[e] - n[e] * s2, dr[e]);
        if constexpr (ADD) as[e] = fmaf(o[i], d[e], as[e]);
      }
      if (a.dx) put_cols<V, AL>(k, a.dx + at.m * a.lddx + at.col, o);
      if constexpr (ADD) {
        if (a.dadd) {
#pragma unroll
          for (int i = 0; i < V; i++) o[i] *= sv[q * V + i];
          put_cols<V, AL>(k, a.dadd + at.m * a.lddadd + at.col, o);
        }
      }
      if constexpr (GATE) {
        if (a.dz) put_cols<V, AL>(k, a.dz + at.m * a.lddz + at.col, z + q * V);
      }
    }
  }
  if (!a.part && !a.dw && !a.dscale) return;
  // the block's groups, added in group order: one access of every lane at a time
  __shared__ float cols[ADD ? 2 : 1][GPB][LPR * V];
#pragma unroll
  for (int q = 0; q < NCH; q++) {
    if (q) __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) {
      cols[0][grp][lr * V + i] = aw[q * V + i];
      if constexpr (ADD) cols[1][grp][lr * V + i] = as[q * V + i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < (ADD ? 2 : 1) * LPR * V; e += kThreads) {
      const int s = e / (LPR * V), l = e % (LPR * V);
      const Cols<V> k((q * LPR + l / V) * V, a.C);
      if (!k.has(l % V)) continue;
      float sum = 0.f;
      for (int i = 0; i < GPB; i++) sum += cols[s][i][l];
      const int col = k.c + l % V;
      if (a.part) a.part[((long)blockIdx.x * 2 + s) * a.C + col] = sum;
      else if (s == 0 && a.dw) a.dw[col] = sum;
      else if (s == 1 && a.dscale) a.dscale[col] = sum;
    }
  }
}

// Rows wider than the registers: a block per row in single elements, two passes; in the gradient a third launch in between adds
// the columns. Bound by the single elements: 16384 rows of 8192 bf16 643 and 1817 us (1.7 and 0.7 TB/s), of 4096, still in registers, 96 and 209.
template <typename T> __device__ __forceinline__ float wide_r(const RmsArgs<T>& a, const At& at, int c) {
  float v, d;
  load_v<1, false>(a.x + at.m * a.ldx + at.col + c, &v);
  if (a.add) {
    load_v<1, false>(a.add + at.m * a.ldadd + at.col + c, &d);
    v = fmaf(a.scale ? a.scale[c] : 1.f, d, v);
  }
  return v;
}
template <typename T> __global__ void __launch_bounds__(kThreads) k_rms_fwd_wide(const RmsArgs<T> a) {
  __shared__ float sh[2][4];
  int turn = 0;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const At at(a, row);
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float v = wide_r(a, at, c);
      s = fmaf(v, v, s);
    }
    const float r = 1.f / sqrtf(row_sum<256>(s, sh, turn) / (float)a.C + a.eps);
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = r;
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float v = wide_r(a, at, c);
      float o = v * r * (a.w ? a.w[c] : 1.f), z;
      if (a.z) {
        load_v<1, false>(a.z + at.m * a.ldz + at.col + c, &z);
        o *= z * sig(z);
      }
      if (a.add && a.res) store_v<1, false>(a.res + at.m * a.ldres + at.col + c, &v);
      store_v<1, false>(a.out + at.m * a.ldout + at.col + c, &o);
    }
  }
}
// One element of a wide row in the gradient: r, n, g = dout silu(z) and (z's own factor) dout silu'(z).
struct WideEl {
  float n, g, gz;
  template <typename T> __device__ __forceinline__ WideEl(const RmsArgs<T>& a, const At& at, long row, int c) {
    n = wide_r(a, at, c) * a.crstd[row];
    load_v<1, false>(a.dout + at.m * a.lddout + at.col + c, &g);
    gz = 0.f;
    if (a.z) {
      float z;
      load_v<1, false>(a.z + at.m * a.ldz + at.col + c, &z);
      const float p = sig(z);
      gz = g * p * fmaf(z, 1.f - p, 1.f);
      g *= z * p;
    }
  }
};
template <typename T> __device__ __forceinline__ float wide_dr(const RmsArgs<T>& a, const At& at, long row, int c, const WideEl& e) {
  float d = 0.f;
  if (a.dres) load_v<1, false>(a.dres + at.m * a.lddres + at.col + c, &d);
  return fmaf(a.crstd[row], e.g * (a.w ? a.w[c] : 1.f) - e.n * a.s2[row], d);
}
template <typename T> __global__ void __launch_bounds__(kThreads) k_rms_bwd_sums_wide(const RmsArgs<T> a) {
  __shared__ float sh[2][4];
  int turn = 0;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const At at(a, row);
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const WideEl e(a, at, row, c);
      s = fmaf(e.g * (a.w ? a.w[c] : 1.f), e.n, s);
    }
    s = row_sum<256>(s, sh, turn) / (float)a.C;
    if (threadIdx.x == 0) a.s2[row] = s;
  }
}
template <typename T> __global__ void __launch_bounds__(kThreads) k_rms_cols_wide(const RmsArgs<T> a) {
  __shared__ float sh[2][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float sw = 0.f, ss = 0.f;
  if (c < a.C)
    for (long row = (long)blockIdx.y * 4 + wave; row < a.rows; row += (long)gridDim.y * 4) {
      const At at(a, row);
      const WideEl e(a, at, row, c);
      sw = fmaf(e.g, e.n, sw);
      if (a.add) {
        float d;
        load_v<1, false>(a.add + at.m * a.ldadd + at.col + c, &d);
        ss = fmaf(wide_dr(a, at, row, c, e), d, ss);
      }
    }
  sh[0][wave][lane] = sw;
  sh[1][wave][lane] = ss;
  __syncthreads();
  if (wave < 2 && c < a.C)
    a.part[((long)blockIdx.y * 2 + wave) * a.C + c] = (sh[wave][0][lane] + sh[wave][1][lane]) + (sh[wave][2][lane] + sh[wave][3][lane]);
}
template <typename T> __global__ void __launch_bounds__(kThreads) k_rms_bwd_wide(const RmsArgs<T> a) {
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const At at(a, row);
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const WideEl e(a, at, row, c);
      const float dr = wide_dr(a, at, row, c, e), dz = e.gz * e.n * (a.w ? a.w[c] : 1.f), dd = dr * (a.scale ? a.scale[c] : 1.f);
      if (a.dx) store_v<1, false>(a.dx + at.m * a.lddx + at.col + c, &dr);
      if (a.add && a.dadd) store_v<1, false>(a.dadd + at.m * a.lddadd + at.col + c, &dd);
      if (a.z && a.dz) store_v<1, false>(a.dz + at.m * a.lddz + at.col + c, &dz);
    }
  }
}
__global__ void k_rms_zero(float* dw, int Cw, float* ds, int C) {
  for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < C; c += gridDim.x * blockDim.x) {
    if (dw && c < Cw) dw[c] = 0.f;
    if (ds) ds[c] = 0.f;
  }
}

// ---- host ------------------------------------------------------------------------------------------
constexpr long kWideBlocks = 1L << 20;

template <typename T> struct RmsCall {
  RmsArgs<T> a;
  bool grad;
  hipStream_t st;

  template <int V, bool AL, int NCH, int LPR, bool ADD, bool GATE> int go() {
    const long per = kThreads / LPR;
    long blocks = (a.rows + per - 1) / per;
    if (!grad) {
      if (blocks > 2048) blocks = 2048;
      k_rms_fwd<T, V, AL, NCH, LPR, ADD, GATE><<<(unsigned)blocks, kThreads, 0, st>>>(a);
      PH_LAUNCH_CHECK();
      return PH_OK;
    }
    // four rows to a group before there are more than 256 blocks: each block's partial row is written, read and added
    long few = (a.rows + 4 * per - 1) / (4 * per);
    if (few < 256) few = blocks < 256 ? blocks : 256;
    blocks = few > 1024 ? 1024 : few;
    a.part = nullptr;
    if (blocks > 1 && (a.dw || a.dscale)) {
      a.part = (float*)scratch(kSlotRms, (size_t)blocks * 2 * a.C * 4);
      if (!a.part) return PH_ERR_NOMEM;
    }
    k_rms_bwd<T, V, AL, NCH, LPR, ADD, GATE><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    PH_LAUNCH_CHECK();
    return fold((int)blocks);
  }
  int fold(int blocks) {
    if (!a.part) return PH_OK;
    const int n = a.dscale ? 2 * a.C : a.C;  // without an add there is no second half
    k_norm_fold<<<(unsigned)((n + 15) / 16), 256, 0, st>>>(a.part, blocks, a.C, a.dw, a.dscale);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  int wide() {
    const unsigned blocks = (unsigned)(a.rows < kWideBlocks ? a.rows : kWideBlocks);
    if (!grad) {
      k_rms_fwd_wide<T><<<blocks, kThreads, 0, st>>>(a);
      PH_LAUNCH_CHECK();
      return PH_OK;
    }
    long ry = (a.rows + 31) / 32;
    if (ry > 128) ry = 128;
    const size_t np = a.dw || a.dscale ? (size_t)ry * 2 * a.C : 0;
    float* ws = (float*)scratch(kSlotRms, (np + (size_t)a.rows) * 4);
    if (!ws) return PH_ERR_NOMEM;
    a.part = np ? ws : nullptr;
    a.s2 = ws + np;
    k_rms_bwd_sums_wide<T><<<blocks, kThreads, 0, st>>>(a);
    PH_LAUNCH_CHECK();
    if (np) {  // before the gradients, which may be written over the inputs
      k_rms_cols_wide<T><<<dim3((a.C + 63) / 64, (unsigned)ry), kThreads, 0, st>>>(a);
      PH_LAUNCH_CHECK();
      PH_TRY(fold((int)ry));
    }
    k_rms_bwd_wide<T><<<blocks, kThreads, 0, st>>>(a);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  template <int V, bool AL, int NCH, int LPR> int by_form() {
    if (a.add) return a.z ? go<V, AL, NCH, LPR, true, true>() : go<V, AL, NCH, LPR, true, false>();
    return a.z ? go<V, AL, NCH, LPR, false, true>() : go<V, AL, NCH, LPR, false, false>();
  }
  template <int V, bool AL> int by_width() {
    const int accesses = (a.C + V - 1) / V;  // of a row
    if (accesses <= 8) return by_form<V, AL, 1, 8>();
    if constexpr (V > 1) {  // fewer columns than a vector access has: one element per lane and access, 8 lanes
      if (accesses <= 16) return by_form<V, AL, 1, 16>();
      if (accesses <= 32) return by_form<V, AL, 1, 32>();
      if (accesses <= 64) return by_form<V, AL, 1, 64>();
      if (accesses <= 128) return by_form<V, AL, 2, 64>();
      if (accesses <= 256) return by_form<V, AL, 1, 256>();
      if (accesses <= 512) return by_form<V, AL, 2, 256>();
    }
    return wide();
  }
  int run() {
    constexpr int V = sizeof(T) == 2 ? 8 : 4;
    if (a.C < V) return by_width<1, false>();
    auto ok = [&](const void* p, long ld) { return !p || (((uintptr_t)p % 16) == 0 && ld % V == 0); };
    const bool al = a.C % V == 0 && ok(a.x, a.ldx) && ok(a.add, a.ldadd) && ok(a.z, a.ldz) && ok(a.out, a.ldout) &&
                    ok(a.res, a.ldres) && ok(a.dout, a.lddout) && ok(a.dres, a.lddres) && ok(a.dx, a.lddx) &&
                    ok(a.dadd, a.lddadd) && ok(a.dz, a.lddz);
    return al ? by_width<V, true>() : by_width<V, false>();
  }
};

int check(const ph_rms_args& p, const char* who) {
  PH_REQUIRE(p.dtype == PH_F32 || p.dtype == PH_BF16, "%s: dtype must be F32 or BF16", who);
  PH_REQUIRE(p.C >= 1 && p.C <= (1u << 20) && p.M <= (1u << 30), "%s: %zu rows of %zu columns", who, p.M, p.C);
  PH_REQUIRE(p.G >= 1 && p.C % p.G == 0 && p.M * p.G <= (1u << 30), "%s: %zu groups of %zu columns, %zu rows", who, p.G, p.C, p.M);
  PH_REQUIRE(!p.scale || ((p.add || p.M == 0) && p.G == 1), "%s: a scale needs an add, and one group", who);
  PH_REQUIRE(p.eps >= 0.f, "%s: eps %g", who, (double)p.eps);
  const long C = (long)p.C;
  PH_REQUIRE(p.ldx >= C && (!p.add || p.ldadd >= C) && (!p.gate || p.ldgate >= C), "%s: a row stride is below %zu columns", who, p.C);
  return PH_OK;
}
// A row is read whole before it is written, by the same lanes: an output may be an input in place, but not lie across one's rows.
struct Rows {
  const void* p;
  long ld;
};
Span span_of(const ph_rms_args& a, const Rows& r) {
  const long e = a.dtype == PH_BF16 ? 2 : 4;
  return {r.p, (long)a.C * e, {(long)a.M, 1, 1}, {r.ld * e, 0, 0}};
}
bool apart(const ph_rms_args& a, const Rows& out, const Rows* in, int n, const float* rstd) {
  for (int i = 0; i < n; i++) {
    const bool same = out.p == in[i].p && (out.ld == in[i].ld || a.M == 1);
    if (!same && meet(span_of(a, out), span_of(a, in[i]))) return false;
  }
  const Span o = span_of(a, out);
  return !meet(o, flat(a.w, (long)(a.C / a.G) * 4)) && !meet(o, flat(a.scale, (long)a.C * 4)) && !meet(o, flat(rstd, (long)(a.M * a.G) * 4));
}
template <typename T> RmsCall<T> call_of(const ph_rms_args& p, void* stream) {
  RmsCall<T> c{};
  RmsArgs<T>& a = c.a;
  a.x = (const T*)p.x; a.add = (const T*)p.add; a.z = (const T*)p.gate;
  a.ldx = p.ldx; a.ldadd = p.ldadd; a.ldz = p.ldgate;
  a.rows = (long)(p.M * p.G);
  a.C = (int)(p.C / p.G); a.G = (int)p.G;
  a.shift = (p.G & (p.G - 1)) == 0 ? __builtin_ctz((unsigned)p.G) : -1;
  a.w = p.w; a.scale = p.scale; a.eps = p.eps;
  c.st = as_stream(stream);
  return c;
}
template <typename T> int fwd_t(const ph_rms_args& p, void* out, long ldout, void* res, long ldres, float* rstd, void* stream) {
  RmsCall<T> c = call_of<T>(p, stream);
  c.a.out = (T*)out; c.a.ldout = ldout; c.a.res = p.add ? (T*)res : nullptr; c.a.ldres = ldres; c.a.rstd = rstd;
  return c.run();
}
template <typename T> int bwd_t(const ph_rms_args& p, const float* rstd, const void* dout, long lddout, const void* dres, long lddres,
                                const ph_rms_grads& g, void* stream) {
  RmsCall<T> c = call_of<T>(p, stream);
  RmsArgs<T>& a = c.a;
  c.grad = true;
  a.crstd = rstd; a.dout = (const T*)dout; a.lddout = lddout; a.dres = (const T*)dres; a.lddres = lddres;
  a.dx = (T*)g.dx; a.lddx = g.lddx; a.dadd = p.add ? (T*)g.dadd : nullptr; a.lddadd = g.lddadd;
  a.dz = p.gate ? (T*)g.dgate : nullptr; a.lddz = g.lddgate;
  a.dw = g.dw; a.dscale = p.scale ? g.dscale : nullptr;
  return c.run();
}

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" int ph_rms_norm(const ph_rms_args* p, void* out, long ldout, void* res, long ldres, float* rstd, void* stream) {
  PH_REQUIRE(p, "rms_norm: arguments missing");
  PH_TRY(check(*p, "rms_norm"));
  const long C = (long)p->C;
  PH_REQUIRE(ldout >= C && (!p->add || !res || ldres >= C), "rms_norm: a row stride is below %zu columns", p->C);
  if (p->M == 0) return PH_OK;
  PH_REQUIRE(p->x && out, "rms_norm: x or out missing");
  const Rows in[] = {{p->x, p->ldx}, {p->add, p->ldadd}, {p->gate, p->ldgate}}, o = {out, ldout}, r = {p->add ? res : nullptr, ldres};
  PH_REQUIRE(!meet(span_of(*p, o), span_of(*p, r)), "rms_norm: out and res are the same or share elements");
  PH_REQUIRE(apart(*p, o, in, 3, rstd) && apart(*p, r, in, 3, rstd), "rms_norm: out or res shares elements with an input that it is not");
  return p->dtype == PH_BF16 ? fwd_t<uint16_t>(*p, out, ldout, res, ldres, rstd, stream)
                             : fwd_t<float>(*p, out, ldout, res, ldres, rstd, stream);
}

extern "C" int ph_rms_norm_grad(const ph_rms_args* p, const float* rstd, const void* dout, long lddout, const void* dres,
                                long lddres, const ph_rms_grads* g, void* stream) {
  PH_REQUIRE(p && g, "rms_norm_grad: arguments missing");
  PH_TRY(check(*p, "rms_norm_grad"));
  const long C = (long)p->C;
  const bool add = p->add && g->dadd, gate = p->gate && g->dgate;
  PH_REQUIRE(lddout >= C && (!dres || lddres >= C) && (!g->dx || g->lddx >= C) && (!add || g->lddadd >= C) && (!gate || g->lddgate >= C),
             "rms_norm_grad: a row stride is below %zu columns", p->C);
  const Rows outs[] = {{g->dx, g->lddx}, {add ? g->dadd : nullptr, g->lddadd}, {gate ? g->dgate : nullptr, g->lddgate}};
  const Rows in[] = {{p->x, p->ldx}, {p->add, p->ldadd}, {p->gate, p->ldgate}, {dout, lddout}, {dres, lddres}};
  for (int i = 0; i < 3; i++)
    for (int j = 0; j < i; j++)
      PH_REQUIRE(!meet(span_of(*p, outs[i]), span_of(*p, outs[j])), "rms_norm_grad: two gradients are the same or share elements");
  for (const Rows& o : outs) PH_REQUIRE(apart(*p, o, in, 5, rstd), "rms_norm_grad: a gradient shares elements with an input that it is not");
  if (p->M == 0) {  // no rows: the columns' sums are zero
    if (!g->dw && !g->dscale) return PH_OK;
    k_rms_zero<<<ceil_div(p->C, 256), 256, 0, as_stream(stream)>>>(g->dw, (int)(p->C / p->G), p->scale ? g->dscale : nullptr, (int)p->C);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  PH_REQUIRE(p->x && dout && rstd, "rms_norm_grad: x, dout or rstd missing");
  return p->dtype == PH_BF16 ? bwd_t<uint16_t>(*p, rstd, dout, lddout, dres, lddres, *g, stream)
                             : bwd_t<float>(*p, rstd, dout, lddout, dres, lddres, *g, stream);
}
