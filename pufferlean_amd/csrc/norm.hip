// Layer normalisation of rows, y = (x - mean) rstd w + b with rstd = 1/sqrt(var + eps), and its gradient.
//
// With n = (x - mean) rstd and dn = dy w, the row's gradient is dx = rstd (dn - avg(dn) - n avg(dn n)); the columns'
// gradients are dw = sum_rows dy n and db = sum_rows dy. All sums are fp32 over values held in registers: the
// variance is the mean of the squared deviations from the row's mean, so a large offset costs no digits.
//
// Both directions are bound by memory: the forward reads x and writes y, the backward reads x and dy and
// writes dx. A row lives in the registers of LPR = 8..64 lanes (64 / LPR rows to a wavefront), so each value
// is read once; the backward's wavefronts walk over many rows and keep their columns' dw and db in registers,
// which leaves one partial row per block for a second, small launch to add in a fixed order.
//
// Measured, 262144 x 512 bf16: forward 103 us and backward 153 us, both 5.2 TB/s, what a large copy reaches on the card,
// and 6 us for the partial rows. 6699 x 203 fp32 (rows of odd width): 5.4, 6.8 and 4.7 us, launch and load latency.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "rows.hpp"

namespace ph {
namespace {

constexpr int kWaves = 4;        // wavefronts per block
constexpr int kNormRegs = 32;    // values of a row that a lane holds at most: rows up to 2048 columns

// V elements per access, NCH accesses per lane: a row has at most LPR * V * NCH columns. A group of LPR lanes walks the
// rows group, group + groups, ... with its columns of w and b in registers: loaded again for every row they cost
// more than the row (262144x512 bf16: 475 us, 103 this way).
template <typename T, int V, bool AL, int NCH, int LPR>
__global__ void __launch_bounds__(64 * kWaves) k_norm_fwd(const T* __restrict__ x, long ldx, long M, int C,
                                                          const float* __restrict__ w, const float* __restrict__ b,
                                                          float eps, T* __restrict__ y, long ldy,
                                                          float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int E = NCH * V, GPB = 64 * kWaves / LPR;
  const int lr = threadIdx.x % LPR;
  float wv[E], bv[E];
#pragma unroll
  for (int q = 0; q < NCH; q++) {
    const Cols<V> k((q * LPR + lr) * V, C);
    get_weights<V>(k, w, 1.f, wv + q * V);
    get_weights<V>(k, b, 0.f, bv + q * V);
  }
  const float inv = 1.f / (float)C;
  // whole groups of LPR lanes leave the loop together; the shuffles stay inside a group
  for (long row = (long)blockIdx.x * GPB + threadIdx.x / LPR; row < M; row += (long)gridDim.x * GPB) {
    float v[E];
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < NCH; q++) get_cols<V, AL>(Cols<V>((q * LPR + lr) * V, C), x + row * ldx, v + q * V);
#pragma unroll
    for (int i = 0; i < E; i++) s += v[i];
    const float mu = group_sum<LPR>(s) * inv;
    float s2 = 0.f;
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      const Cols<V> k((q * LPR + lr) * V, C);
#pragma unroll
      for (int i = 0; i < V; i++) {
        v[q * V + i] -= mu;
        s2 += (AL ? k.in : k.has(i)) ? v[q * V + i] * v[q * V + i] : 0.f;
      }
    }
    const float r = 1.f / sqrtf(group_sum<LPR>(s2) * inv + eps);
    if (lr == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; i++) o[i] = fmaf(v[q * V + i] * r, wv[q * V + i], bv[q * V + i]);
      put_cols<V, AL>(Cols<V>((q * LPR + lr) * V, C), y + row * ldy, o);
    }
  }
}

// Rows wider than the registers: one block per row, three passes over it in single elements; in the gradient two, behind one of
// k_norm_cols_wide. 65536 x 2056 forward and gradient bf16 416 and 577 us, fp32 488 and 696 (2048 columns in
// registers: 111 and 216, 184 and 291); 64 x 4096 take the host's call. A launch of 2^32 threads or more would start the
// remainder only, so past kWideBlocks rows a block goes on to its next ones.
constexpr long kWideBlocks = 1L << 20;
template <typename T>
__global__ void __launch_bounds__(256) k_norm_fwd_wide(const T* __restrict__ x, long ldx, long M, int C,
                                                       const float* __restrict__ w, const float* __restrict__ b,
                                                       float eps, T* __restrict__ y, long ldy,
                                                       float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float sh[2][4];
  auto total = [&](float v, int k) {
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) sh[k][threadIdx.x >> 6] = v;
    __syncthreads();
    return (sh[k][0] + sh[k][1]) + (sh[k][2] + sh[k][3]);
  };
  // a row's two sums have buffers of their own, so between reading one and writing it again there is the other's barrier
  for (long row = blockIdx.x; row < M; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float v, s = 0.f;
    for (int c = threadIdx.x; c < C; c += 256) {
      load_v<1, false>(xr + c, &v);
      s += v;
    }
    const float mu = total(s, 0) / (float)C;
    s = 0.f;
    for (int c = threadIdx.x; c < C; c += 256) {
      load_v<1, false>(xr + c, &v);
      s += (v - mu) * (v - mu);
    }
    const float r = 1.f / sqrtf(total(s, 1) / (float)C + eps);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = mu;
      if (rstd) rstd[row] = r;
    }
    for (int c = threadIdx.x; c < C; c += 256) {
      load_v<1, false>(xr + c, &v);
      v = (v - mu) * r * (w ? w[c] : 1.f) + (b ? b[c] : 0.f);
      store_v<1, false>(y + row * ldy + c, &v);
    }
  }
}

// Backward: a group of LPR lanes walks the rows group, group + groups, ...; dw and db of its columns stay in its
// registers and are added over the block's groups through LDS. part: [blocks][2][C] (or dw, db themselves for one block).
template <typename T, int V, bool AL, int NCH, int LPR>
__global__ void __launch_bounds__(64 * kWaves) k_norm_bwd(const T* __restrict__ x, long ldx, const T* __restrict__ dy,
                                                          long lddy, long M, int C, const float* __restrict__ w,
                                                          const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, T* __restrict__ dx,
                                                          long lddx, float* __restrict__ dw, float* __restrict__ db,
                                                          float* __restrict__ part) {
  constexpr int E = NCH * V, GPB = 64 * kWaves / LPR;
  static_assert(E <= kNormRegs, "registers of a row");
  const int lr = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  float aw[E], ab[E], wv[E];
#pragma unroll
  for (int q = 0; q < NCH; q++) {
    get_weights<V>(Cols<V>((q * LPR + lr) * V, C), w, 1.f, wv + q * V);
#pragma unroll
    for (int i = 0; i < V; i++) aw[q * V + i] = ab[q * V + i] = 0.f;
  }
  const float inv = 1.f / (float)C;
  for (long row = (long)blockIdx.x * GPB + grp; row < M; row += (long)gridDim.x * GPB) {
    float n[E], g[E];
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      const Cols<V> k((q * LPR + lr) * V, C);
      get_cols<V, AL>(k, x + row * ldx, n + q * V);
      get_cols<V, AL>(k, dy + row * lddy, g + q * V);
    }
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) {
      n[i] = (n[i] - mu) * r;
      aw[i] += g[i] * n[i];  // dy is zero where the lane has no column
      ab[i] += g[i];
      g[i] *= wv[i];
      s1 += g[i];
      s2 += g[i] * n[i];
    }
    group_sum<LPR>(s1, s2);
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int q = 0; q < NCH; q++) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; i++) o[i] = r * (g[q * V + i] - s1 - n[q * V + i] * s2);
      put_cols<V, AL>(Cols<V>((q * LPR + lr) * V, C), dx + row * lddx, o);
    }
  }
  if (!part && !dw && !db) return;
  // the block's groups, added in group order: one access of every lane at a time
  __shared__ float sh[2][GPB][LPR * V];
#pragma unroll
  for (int q = 0; q < NCH; q++) {
    if (q) __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) {
      sh[0][grp][lr * V + i] = aw[q * V + i];
      sh[1][grp][lr * V + i] = ab[q * V + i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * LPR * V; e += 64 * kWaves) {
      const int s = e / (LPR * V), l = e % (LPR * V);
      const Cols<V> k((q * LPR + l / V) * V, C);
      if (!k.has(l % V)) continue;
      float sum = 0.f;
      for (int i = 0; i < GPB; i++) sum += sh[s][i][l];
      const int col = k.c + l % V;
      if (part) part[((long)blockIdx.x * 2 + s) * C + col] = sum;
      else if (s == 0 && dw) dw[col] = sum;
      else if (s == 1 && db) db[col] = sum;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_norm_bwd_wide(const T* __restrict__ x, long ldx, const T* __restrict__ dy,
                                                       long lddy, long M, int C, const float* __restrict__ w,
                                                       const float* __restrict__ mean, const float* __restrict__ rstd,
                                                       T* __restrict__ dx, long lddx) {
  __shared__ float sh[2][2][4];  // of alternate rows: every thread has read a row's in front of the next one's barrier
  int p = 0;
  for (long row = blockIdx.x; row < M; row += gridDim.x, p ^= 1) {
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f, a, g;
    for (int c = threadIdx.x; c < C; c += 256) {
      load_v<1, false>(x + row * ldx + c, &a);
      load_v<1, false>(dy + row * lddy + c, &g);
      g *= w ? w[c] : 1.f;
      s1 += g;
      s2 += g * (a - mu) * r;
    }
    s1 = group_sum<64>(s1);
    s2 = group_sum<64>(s2);
    if ((threadIdx.x & 63) == 0) {
      sh[p][0][threadIdx.x >> 6] = s1;
      sh[p][1][threadIdx.x >> 6] = s2;
    }
    __syncthreads();
    s1 = ((sh[p][0][0] + sh[p][0][1]) + (sh[p][0][2] + sh[p][0][3])) / (float)C;
    s2 = ((sh[p][1][0] + sh[p][1][1]) + (sh[p][1][2] + sh[p][1][3])) / (float)C;
    for (int c = threadIdx.x; c < C; c += 256) {
      load_v<1, false>(x + row * ldx + c, &a);
      load_v<1, false>(dy + row * lddy + c, &g);
      a = r * (g * (w ? w[c] : 1.f) - s1 - (a - mu) * r * s2);
      store_v<1, false>(dx + row * lddx + c, &a);
    }
  }
}
// dw and db partials of wide rows: 64 columns x a range of rows per block of four wavefronts.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_cols_wide(const T* __restrict__ x, long ldx, const T* __restrict__ dy,
                                                        long lddy, long M, int C, const float* __restrict__ mean,
                                                        const float* __restrict__ rstd, float* __restrict__ part) {
  __shared__ float sh[2][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float sw = 0.f, sb = 0.f, a, g;
  if (c < C)
    for (long row = (long)blockIdx.y * 4 + wave; row < M; row += (long)gridDim.y * 4) {
      load_v<1, false>(x + row * ldx + c, &a);
      load_v<1, false>(dy + row * lddy + c, &g);
      sw += g * (a - mean[row]) * rstd[row];
      sb += g;
    }
  sh[0][wave][lane] = sw;
  sh[1][wave][lane] = sb;
  __syncthreads();
  if (wave < 2 && c < C)
    part[((long)blockIdx.y * 2 + wave) * C + c] = (sh[wave][0][lane] + sh[wave][1][lane]) + (sh[wave][2][lane] + sh[wave][3][lane]);
}

__global__ void k_norm_zero(float* dw, float* db, int C) {
  for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < C; c += gridDim.x * blockDim.x) {
    if (dw) dw[c] = 0.f;
    if (db) db[c] = 0.f;
  }
}

// One call's arguments, and its dispatch over (V, NCH, LPR).
template <typename T> struct NormCall {
  const T *x, *dy;
  T *y, *dx;
  long ldx, lddy, ldy, lddx, M;
  int C;
  const float *w, *b;
  float eps;
  float *mean, *rstd;
  const float *cmean, *crstd;
  float *dw, *db;
  hipStream_t st;

  template <int V, bool AL, int NCH, int LPR> int forward() const {
    const long rows = 64 * kWaves / LPR;
    long blocks = (M + rows - 1) / rows;
    const long most = NCH * V > 8 ? 1024 : 2048;  // as many as run at a time: rows of 512 columns and more take more registers
    if (blocks > most) blocks = most;
    k_norm_fwd<T, V, AL, NCH, LPR><<<(unsigned)blocks, 64 * kWaves, 0, st>>>(x, ldx, M, C, w, b, eps, y, ldy, mean, rstd);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  template <int V, bool AL, int NCH, int LPR> int backward() const {
    const long rows = 64 * kWaves / LPR;
    // four rows to a group before there are more than 256 blocks: each block's partial row is written, read and added
    long blocks = (M + 4 * rows - 1) / (4 * rows);
    if (blocks < 256) blocks = (M + rows - 1) / rows < 256 ? (M + rows - 1) / rows : 256;
    if (blocks > 1024) blocks = 1024;
    float* part = nullptr;
    if (blocks > 1 && (dw || db)) {
      part = (float*)scratch(kSlotNormPart, (size_t)blocks * 2 * C * 4);
      if (!part) return PH_ERR_NOMEM;
    }
    k_norm_bwd<T, V, AL, NCH, LPR><<<(unsigned)blocks, 64 * kWaves, 0, st>>>(x, ldx, dy, lddy, M, C, w, cmean, crstd, dx,
                                                                         lddx, dw, db, part);
    PH_LAUNCH_CHECK();
    if (part) {
      k_norm_fold<<<(unsigned)((2 * C + 15) / 16), 256, 0, st>>>(part, (int)blocks, C, dw, db);
      PH_LAUNCH_CHECK();
    }
    return PH_OK;
  }
  template <int V, bool AL, int NCH, int LPR> int go() const { return dy ? backward<V, AL, NCH, LPR>() : forward<V, AL, NCH, LPR>(); }
  int wide() const {
    const unsigned blocks = (unsigned)(M < kWideBlocks ? M : kWideBlocks);
    if (!dy) {
      k_norm_fwd_wide<T><<<blocks, 256, 0, st>>>(x, ldx, M, C, w, b, eps, y, ldy, mean, rstd);
      PH_LAUNCH_CHECK();
      return PH_OK;
    }
    // the columns' sums first: dx may be written over x or dy
    if (dw || db) {
      long ry = (M + 31) / 32;
      if (ry > 128) ry = 128;
      float* part = (float*)scratch(kSlotNormPart, (size_t)ry * 2 * C * 4);
      if (!part) return PH_ERR_NOMEM;
      k_norm_cols_wide<T><<<dim3((C + 63) / 64, (unsigned)ry), 256, 0, st>>>(x, ldx, dy, lddy, M, C, cmean, crstd, part);
      PH_LAUNCH_CHECK();
      k_norm_fold<<<(unsigned)((2 * C + 15) / 16), 256, 0, st>>>(part, (int)ry, C, dw, db);
      PH_LAUNCH_CHECK();
    }
    k_norm_bwd_wide<T><<<blocks, 256, 0, st>>>(x, ldx, dy, lddy, M, C, w, cmean, crstd, dx, lddx);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  template <int V, bool AL> int by_width() const {
    const int accesses = (C + V - 1) / V;  // of a row
    if (accesses <= 8) return go<V, AL, 1, 8>();
    if constexpr (V > 1) {  // fewer columns than a vector access has: one element per lane and access, 8 lanes
      if (accesses <= 16) return go<V, AL, 1, 16>();
      if (accesses <= 32) return go<V, AL, 1, 32>();
      if (accesses <= 64) return go<V, AL, 1, 64>();
      if (accesses <= 128) return go<V, AL, 2, 64>();
      if (accesses <= 256) return go<V, AL, 4, 64>();
      if constexpr (8 * V <= kNormRegs) {
        if (accesses <= 512) return go<V, AL, 8, 64>();
      }
    }
    return wide();
  }
  int run() const {
    constexpr int V = sizeof(T) == 2 ? 8 : 4;
    if (C < V) return by_width<1, false>();
    auto ok = [&](const void* p, long ld) { return !p || (((uintptr_t)p % 16) == 0 && ld % V == 0); };
    const bool al = C % V == 0 && ok(x, ldx) && ok(y, ldy) && ok(dy, lddy) && ok(dx, lddx);
    return al ? by_width<V, true>() : by_width<V, false>();
  }
};

template <typename T> int norm_fwd_t(const void* x, size_t ldx, size_t M, size_t C, const float* w, const float* b,
                                     float eps, void* y, size_t ldy, float* mean, float* rstd, hipStream_t st) {
  NormCall<T> c{};
  c.x = (const T*)x; c.y = (T*)y; c.ldx = (long)ldx; c.ldy = (long)ldy; c.M = (long)M; c.C = (int)C;
  c.w = w; c.b = b; c.eps = eps; c.mean = mean; c.rstd = rstd; c.st = st;
  return c.run();
}
template <typename T> int norm_bwd_t(const void* x, size_t ldx, const void* dy, size_t lddy, size_t M, size_t C,
                                     const float* w, const float* mean, const float* rstd, void* dx, size_t lddx,
                                     float* dw, float* db, hipStream_t st) {
  NormCall<T> c{};
  c.x = (const T*)x; c.dy = (const T*)dy; c.dx = (T*)dx; c.ldx = (long)ldx; c.lddy = (long)lddy; c.lddx = (long)lddx;
  c.M = (long)M; c.C = (int)C; c.w = w; c.cmean = mean; c.crstd = rstd; c.dw = dw; c.db = db; c.st = st;
  return c.run();
}

constexpr size_t kNormMaxCols = 1u << 20;
constexpr size_t kNormMaxRows = 1u << 30;

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" int ph_layer_norm(int dtype, const void* x, size_t ldx, size_t M, size_t C, const float* w, const float* b,
                             float eps, void* y, size_t ldy, float* mean, float* rstd, void* stream) {
  PH_REQUIRE(dtype == PH_F32 || dtype == PH_BF16, "layer_norm: dtype must be F32 or BF16");
  PH_REQUIRE(C >= 1 && C <= kNormMaxCols && M <= kNormMaxRows, "layer_norm: %zu rows of %zu columns", M, C);
  PH_REQUIRE(ldx >= C && ldy >= C, "layer_norm: row strides %zu, %zu below %zu columns", ldx, ldy, C);
  PH_REQUIRE(eps >= 0.f, "layer_norm: eps %g", (double)eps);
  if (M == 0) return PH_OK;
  PH_REQUIRE(x && y, "layer_norm: x or y missing");
  return dtype == PH_BF16 ? norm_fwd_t<uint16_t>(x, ldx, M, C, w, b, eps, y, ldy, mean, rstd, as_stream(stream))
                          : norm_fwd_t<float>(x, ldx, M, C, w, b, eps, y, ldy, mean, rstd, as_stream(stream));
}

extern "C" int ph_layer_norm_grad(int dtype, const void* x, size_t ldx, const void* dy, size_t lddy, size_t M, size_t C,
                                  const float* w, const float* mean, const float* rstd, void* dx, size_t lddx,
                                  float* dw, float* db, void* stream) {
  PH_REQUIRE(dtype == PH_F32 || dtype == PH_BF16, "layer_norm_grad: dtype must be F32 or BF16");
  PH_REQUIRE(C >= 1 && C <= kNormMaxCols && M <= kNormMaxRows, "layer_norm_grad: %zu rows of %zu columns", M, C);
  PH_REQUIRE(ldx >= C && lddy >= C && lddx >= C, "layer_norm_grad: a row stride is below %zu columns", C);
  if (M == 0) {  // no rows: the columns' sums are zero
    if (!dw && !db) return PH_OK;
    k_norm_zero<<<ceil_div(C, 256), 256, 0, as_stream(stream)>>>(dw, db, (int)C);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  PH_REQUIRE(x && dy && dx && mean && rstd, "layer_norm_grad: x, dy, dx, mean or rstd missing");
  return dtype == PH_BF16 ? norm_bwd_t<uint16_t>(x, ldx, dy, lddy, M, C, w, mean, rstd, dx, lddx, dw, db, as_stream(stream))
                          : norm_bwd_t<float>(x, ldx, dy, lddy, M, C, w, mean, rstd, dx, lddx, dw, db, as_stream(stream));
}
