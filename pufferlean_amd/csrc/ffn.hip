// Gated feed-forward block y = (act(x Wg^T) * (x Wv^T)) Wo^T and its gradient. With the projections a = x Wg^T and
// v = x Wv^T interleaved in the columns of x w_in^T, h = act(a) v:
//
//   forward   h, p = v act'(a), f = act(a) from one product x w_in^T;  y = h w_out^T
//   backward  dab = (dh p, dh f) interleaved, from one product dh = dy w_out;
//             dw_out = dy^T h;  dw_in = dab^T x;  dx = dab w_in
//
// All on the matrix cores: 6 M D F operations forward and 12 M D F backward, against which the activations' traffic is
// small; the epilogues (glu.hpp) keep the projections and dh from ever being written. bf16 rounds h, p, f and dab once
// each from fp32: they are the operands of bf16 products, or (p, f) halve what the backward reads.
//
// The products want whole 16-byte accesses. Where D or F is not a multiple of 8, or a pointer or stride is off, the inputs'
// rows and the weights are copied once, padded with zeros, which add nothing to any sum.
#include "common.hpp"
#include "glu.hpp"
#include "kernels.hpp"

#include <type_traits>

namespace ph {
namespace {

size_t up8(size_t n) { return (n + 7) / 8 * 8; }

// One copy: dst [rows_p][cols_p] = src [rows][cols] (row stride ld) with zeros beyond, or its transpose, [cols_p][rows_p].
struct Lay {
  const void* src;
  void* dst;
  long rows, cols, ld, rows_p, cols_p;
  int trans;
  unsigned first;  // block of its first 32 x 32 tile
};
constexpr int kMostLays = 4;
struct Lays {
  Lay l[kMostLays];
  int n;
  unsigned blocks;
};
// All copies of a call in one launch, a 32 x 32 tile per block.
template <typename T>
__global__ void __launch_bounds__(256) k_lay(Lays ls) {
  __shared__ T tile[32][33];
  int w = 0;
  while (w + 1 < ls.n && blockIdx.x >= ls.l[w + 1].first) w++;
  const Lay& j = ls.l[w];
  const T* src = (const T*)j.src;
  T* dst = (T*)j.dst;
  const long nc = (j.cols_p + 31) / 32, id = blockIdx.x - j.first, r0 = id / nc * 32, c0 = id % nc * 32;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const long r = r0 + y + i, c = c0 + x;
    const T v = r < j.rows && c < j.cols ? src[r * j.ld + c] : T(0);
    if (!j.trans) {
      if (r < j.rows_p && c < j.cols_p) dst[r * j.cols_p + c] = v;
    } else {
      tile[y + i][x] = v;
    }
  }
  if (!j.trans) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const long c = c0 + y + i, r = r0 + x;
    if (r < j.rows_p && c < j.cols_p) dst[c * j.rows_p + r] = tile[x][y + i];
  }
}

// Collects a call's copies.
struct Layer {
  Lays ls{};
  int add(const void* src, size_t rows, size_t cols, size_t ld, void* dst, size_t rows_p, size_t cols_p, bool trans) {
    const size_t blocks = ls.blocks + (rows_p + 31) / 32 * ((cols_p + 31) / 32);
    PH_REQUIRE(blocks < (1u << 31) && ls.n < kMostLays, "ffn: %zu x %zu values to lay out", rows_p, cols_p);
    ls.l[ls.n++] = Lay{src, dst, (long)rows, (long)cols, (long)ld, (long)rows_p, (long)cols_p, trans, ls.blocks};
    ls.blocks = (unsigned)blocks;
    return PH_OK;
  }
  int run(int dtype, hipStream_t st) {
    if (!ls.n) return PH_OK;
    if (dtype == PH_BF16) k_lay<uint16_t><<<ls.blocks, 256, 0, st>>>(ls);
    else k_lay<float><<<ls.blocks, 256, 0, st>>>(ls);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
};

// ---- few rows --------------------------------------------------------------------------------------------
// Up to 64 rows are bound by the weights' bytes and by latency, so the weights go from memory straight into the operand
// registers of 16x16x32 products (16 weight rows to a wavefront, a lane 8 consecutive values of one), with the
// rows of x as the other operand; the block's wavefronts share the reduction and are added through LDS.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
constexpr int kFewRows = 64;

__device__ __forceinline__ bf16x8_t frag(const uint16_t* row, long k, long K) {
  const uint4 v = k < K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0u, 0u, 0u, 0u);
  return __builtin_bit_cast(bf16x8_t, v);
}
// acc[m][r] = the products of weight rows w0 + 4 (lane / 16) + r and x rows 16 m + lane % 16 over this wavefront's share
// of k, then summed over the block's WAVES wavefronts: wavefront m < MT returns with block m's in acc[0].
template <int MT, int WAVES>
__device__ __forceinline__ void few_rows(f32x4_t (&acc)[MT], const uint16_t* w, long ldw, int w0, int wrows, const uint16_t* x,
                                         long ldx, int M, long K, float* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15;
  const uint16_t* wr = w + (long)min(w0 + r, wrows - 1) * ldw;
  const uint16_t* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    xr[m] = x + (long)min(16 * m + r, M - 1) * ldx;  // rows past M repeat the last; they are not stored
    acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const long steps = (K + 31) / 32, per = (steps + WAVES - 1) / WAVES, beg = wave * per, end = min(steps, beg + per);
  const int ko = 8 * (lane >> 4);
#pragma unroll 4
  for (long s = beg; s < end; s++) {
    const bf16x8_t a = frag(wr, 32 * s + ko, K);
#pragma unroll
    for (int m = 0; m < MT; m++)
      acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, frag(xr[m], 32 * s + ko, K), acc[m], 0, 0, 0);
  }
  f32x4_t* sh = reinterpret_cast<f32x4_t*>(red);  // [WAVES][MT][64]
#pragma unroll
  for (int m = 0; m < MT; m++) sh[(wave * MT + m) * 64 + lane] = acc[m];
  __syncthreads();
  if (wave >= MT) return;
  f32x4_t s = sh[wave * 64 + lane];
  for (int v = 1; v < WAVES; v++) s += sh[(v * MT + wave) * 64 + lane];
  acc[0] = s;
}

template <int MT>
__global__ void __launch_bounds__(256) k_few_in(const uint16_t* __restrict__ x, long ldx, const uint16_t* __restrict__ w, long D,
                                                int M, int F, int act, uint16_t* __restrict__ h, uint16_t* __restrict__ pf) {
  __shared__ __attribute__((aligned(16))) float red[4 * MT * 64 * 4];
  f32x4_t acc[MT];
  few_rows<MT, 4>(acc, w, D, blockIdx.x * 16, 2 * F, x, ldx, M, D, red);
  const int lane = threadIdx.x & 63, row = 16 * (threadIdx.x >> 6) + (lane & 15), u = blockIdx.x * 8 + 2 * (lane >> 4);
  if ((threadIdx.x >> 6) >= MT || row >= M) return;
  float f0, d0, f1, d1;
  glu_act(act, acc[0][0], f0, d0);
  glu_act(act, acc[0][2], f1, d1);
  *reinterpret_cast<uint32_t*>(h + (long)row * F + u) = bf16x2_rne(f0 * acc[0][1], f1 * acc[0][3]);
  if (pf)
    *reinterpret_cast<uint2*>(pf + (long)row * 2 * F + 2 * u) =
        make_uint2(bf16x2_rne(acc[0][1] * d0, f0), bf16x2_rne(acc[0][3] * d1, f1));
}

template <int MT>
__global__ void __launch_bounds__(512) k_few_out(const uint16_t* __restrict__ h, const uint16_t* __restrict__ w, long F, int M, int D,
                                                 uint16_t* __restrict__ y, long ldy) {
  __shared__ __attribute__((aligned(16))) float red[8 * MT * 64 * 4];
  f32x4_t acc[MT];
  few_rows<MT, 8>(acc, w, F, blockIdx.x * 16, D, h, F, M, F, red);
  const int lane = threadIdx.x & 63, row = 16 * (threadIdx.x >> 6) + (lane & 15), d = blockIdx.x * 16 + 4 * (lane >> 4);
  if ((threadIdx.x >> 6) >= MT || row >= M) return;
#pragma unroll
  for (int r = 0; r < 4; r++)
    if (d + r < D) y[(long)row * ldy + d + r] = bf16_rne(acc[0][r]);
}

template <int MT>
int few_rows_ffn(const uint16_t* x, long ldx, const uint16_t* w_in, const uint16_t* w_out, int M, int D, int F, int act,
                 uint16_t* h, uint16_t* pf, uint16_t* y, long ldy, hipStream_t st) {
  k_few_in<MT><<<(unsigned)(2 * F / 16), 256, 0, st>>>(x, ldx, w_in, D, M, F, act, h, pf);
  PH_LAUNCH_CHECK();
  k_few_out<MT><<<(unsigned)((D + 15) / 16), 512, 0, st>>>(h, w_out, F, M, D, y, ldy);
  PH_LAUNCH_CHECK();
  return PH_OK;
}

int product(int ta, int tb, size_t M, size_t N, size_t K, int dtype, const void* A, size_t lda, const void* B, size_t ldb,
            int c_dtype, void* C, size_t ldc, hipStream_t st) {
  PhGemmDesc d{};
  d.trans_a = ta; d.trans_b = tb; d.M = (int)M; d.N = (int)N; d.K = (int)K;
  d.a_dtype = d.b_dtype = dtype; d.A = A; d.lda = (long)lda; d.B = B; d.ldb = (long)ldb;
  d.c_dtype = c_dtype; d.C = C; d.ldc = (long)ldc;
  d.math = dtype == PH_BF16 ? PH_MATH_BF16 : PH_MATH_F32;
  return gemm(d, st);
}

// Rows from which the backward's products take transposed weights.
constexpr size_t kTransposeRows = 2048;

// One call's sizes, and its scratch handed out in pieces of 256 bytes.
struct Call {
  int dtype, act;
  size_t M, D, F, Dp, Fp, e;
  hipStream_t st;
  uint8_t* ws = nullptr;
  size_t need = 0, used = 0;

  Call(int dt, int ac, size_t m, size_t d, size_t f, hipStream_t s)
      : dtype(dt), act(ac), M(m), D(d), F(f), Dp(up8(d)), Fp(up8(f)), e(dt == PH_BF16 ? 2 : 4), st(s) {}
  static size_t round(size_t bytes) { return (bytes + 255) / 256 * 256; }
  void want(size_t elements, size_t size) { need += round(elements * size); }
  int take_all() {
    ws = need ? (uint8_t*)scratch(kSlotFfn, need) : nullptr;
    return need && !ws ? PH_ERR_NOMEM : PH_OK;
  }
  void* take(size_t elements, size_t size) {
    void* p = ws + used;
    used += round(elements * size);
    return p;
  }
  // Whether rows of `cols` values at p can be read as they are: whole 16-byte accesses, `cols` being its padded width.
  bool whole(const void* p, size_t ld, size_t cols, size_t padded) const {
    return cols == padded && ld % 8 == 0 && ((uintptr_t)p % 16) == 0;
  }
  int check(const char* who) const {
    PH_REQUIRE(dtype == PH_F32 || dtype == PH_BF16, "%s: dtype must be F32 or BF16", who);
    PH_REQUIRE(act == PH_ACT_SILU || act == PH_ACT_GELU, "%s: unknown activation %d", who, act);
    PH_REQUIRE(D >= 1 && F >= 1 && D <= (1u << 20) && F <= (1u << 20) && M <= (1u << 30), "%s: M = %zu, D = %zu, F = %zu out of range",
               who, M, D, F);
    return PH_OK;
  }
};

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" size_t ph_ffn_pitch(size_t columns) { return up8(columns); }

extern "C" int ph_ffn(int dtype, int act, size_t M, size_t D, size_t F, const void* x, size_t ldx, const void* w_in,
                      const void* w_out, void* pf, void* h, void* y, size_t ldy, void* stream) {
  Call c(dtype, act, M, D, F, as_stream(stream));
  PH_TRY(c.check("ffn"));
  PH_REQUIRE(ldx >= D && ldy >= D, "ffn: row strides %zu, %zu below %zu columns", ldx, ldy, D);
  if (M == 0) return PH_OK;
  PH_REQUIRE(x && w_in && w_out && y, "ffn: x, w_in, w_out or y missing");
  PH_REQUIRE(!pf == !h, "ffn: pf and h are kept together");
  const size_t Dp = c.Dp, Fp = c.Fp;
  const bool x_ok = c.whole(x, ldx, D, Dp), wi_ok = F == Fp && c.whole(w_in, D, D, Dp), wo_ok = c.whole(w_out, F, F, Fp);
  if (!x_ok) c.want(M * Dp, c.e);
  if (!wi_ok) c.want(2 * Fp * Dp, c.e);
  if (!wo_ok) c.want(D * Fp, c.e);
  if (!h) c.want(M * Fp, c.e);
  PH_TRY(c.take_all());
  Layer lay;
  auto padded = [&](const void*& p, size_t rows, size_t cols, size_t ld, size_t rows_p, size_t cols_p) {
    void* q = c.take(rows_p * cols_p, c.e);
    const void* src = p;
    p = q;
    return lay.add(src, rows, cols, ld, q, rows_p, cols_p, false);
  };
  if (!x_ok) {
    PH_TRY(padded(x, M, D, ldx, M, Dp));
    ldx = Dp;
  }
  if (!wi_ok) PH_TRY(padded(w_in, 2 * F, D, D, 2 * Fp, Dp));
  if (!wo_ok) PH_TRY(padded(w_out, D, F, F, D, Fp));
  PH_TRY(lay.run(dtype, c.st));
  if (!h) h = c.take(M * Fp, c.e);
  if (dtype == PH_BF16 && M <= (size_t)kFewRows && F == Fp) {
    auto run = [&](auto mt) {
      return few_rows_ffn<decltype(mt)::value>((const uint16_t*)x, (long)ldx, (const uint16_t*)w_in, (const uint16_t*)w_out, (int)M,
                                               (int)D, (int)F, act, (uint16_t*)h, (uint16_t*)pf, (uint16_t*)y, (long)ldy, c.st);
    };
    if (D == Dp) {
      if (M <= 16) return run(std::integral_constant<int, 1>{});
      if (M <= 32) return run(std::integral_constant<int, 2>{});
      return run(std::integral_constant<int, 4>{});
    }
  }
  GluProduct g{};
  g.dtype = dtype; g.act = act; g.M = (int)M; g.N = (int)(2 * Fp); g.K = (int)Dp;
  g.A = x; g.lda = (long)ldx; g.B = w_in; g.ldb = (long)Dp; g.h = h; g.ldh = (long)Fp; g.pf = pf; g.ldpf = (long)(2 * Fp);
  PH_TRY(glu_product(g, c.st));
  return product(0, 1, M, D, Fp, dtype, h, Fp, w_out, Fp, dtype, y, ldy, c.st);
}

extern "C" int ph_ffn_grad(int dtype, int act, size_t M, size_t D, size_t F, const void* x, size_t ldx, const void* w_in,
                           const void* w_out, const void* pf, const void* h, const void* dy, size_t lddy, void* dx,
                           size_t lddx, int dw_dtype, void* dw_in, void* dw_out, void* stream) {
  Call c(dtype, act, M, D, F, as_stream(stream));
  PH_TRY(c.check("ffn_grad"));
  PH_REQUIRE(dw_dtype == dtype || dw_dtype == PH_F32, "ffn_grad: the weights' gradients are of dtype or F32");
  PH_REQUIRE(ldx >= D && lddy >= D && (!dx || lddx >= D), "ffn_grad: a row stride is below %zu columns", D);
  PH_REQUIRE(M == 0 || (x && w_in && w_out && pf && h && dy), "ffn_grad: an input is missing");
  if (M == 0) {  // no rows: the weights' sums are zero
    if (dw_in) PH_TRY(product(1, 0, 2 * F, D, 0, dtype, nullptr, c.Fp, nullptr, c.Dp, dw_dtype, dw_in, D, c.st));
    if (dw_out) PH_TRY(product(1, 0, D, F, 0, dtype, nullptr, c.Dp, nullptr, c.Fp, dw_dtype, dw_out, F, c.st));
    return PH_OK;
  }
  const size_t Dp = c.Dp, Fp = c.Fp, we = dw_dtype == PH_BF16 ? 2 : 4;
  const bool x_ok = c.whole(x, ldx, D, Dp), dy_ok = c.whole(dy, lddy, D, Dp), w_ok = D == Dp && F == Fp;
  // Transposed copies of the weights, so that both products read their operands along k: with many rows the products
  // are faster by more than the copies take. With few rows the products take the weights as they are (or padded).
  const bool trans = M >= kTransposeRows;
  const bool wo_ok = !trans && c.whole(w_out, F, F, Fp) && D == Dp, wi_ok = !trans && c.whole(w_in, D, D, Dp) && F == Fp;
  const bool need_dab = dx || dw_in;
  if (!x_ok && dw_in) c.want(M * Dp, c.e);
  if (!dy_ok) c.want(M * Dp, c.e);
  if (need_dab) {
    if (!wo_ok) c.want(Fp * Dp, c.e);
    if (!wi_ok && dx) c.want(2 * Fp * Dp, c.e);
    c.want(M * 2 * Fp, c.e);
  }
  if (!w_ok) c.want(2 * Fp * Dp, we), c.want(Fp * Dp, we);
  PH_TRY(c.take_all());
  Layer lay;
  auto laid = [&](const void*& p, size_t rows, size_t cols, size_t ld, size_t rows_p, size_t cols_p, bool tr) {
    void* q = c.take(rows_p * cols_p, c.e);
    const void* src = p;
    p = q;
    return lay.add(src, rows, cols, ld, q, rows_p, cols_p, tr);
  };
  if (!x_ok && dw_in) {
    PH_TRY(laid(x, M, D, ldx, M, Dp, false));
    ldx = Dp;
  }
  if (!dy_ok) {
    PH_TRY(laid(dy, M, D, lddy, M, Dp, false));
    lddy = Dp;
  }
  void* dab = nullptr;
  if (need_dab) {
    if (!wo_ok) PH_TRY(laid(w_out, D, F, F, Dp, Fp, trans));
    if (!wi_ok && dx) PH_TRY(laid(w_in, 2 * F, D, D, 2 * Fp, Dp, trans));
    dab = c.take(M * 2 * Fp, c.e);
  }
  PH_TRY(lay.run(dtype, c.st));
  if (need_dab) {
    GluProduct g{};
    g.grad = 1; g.dtype = dtype; g.act = act; g.M = (int)M; g.N = (int)Fp; g.K = (int)Dp; g.b_kn = !trans;
    g.A = dy; g.lda = (long)lddy; g.B = w_out; g.ldb = (long)(trans ? Dp : Fp);
    g.pf = const_cast<void*>(pf); g.ldpf = (long)(2 * Fp); g.dab = dab; g.lddab = (long)(2 * Fp);
    PH_TRY(glu_product(g, c.st));
  }
  if (dx) PH_TRY(product(0, trans, M, D, 2 * Fp, dtype, dab, 2 * Fp, w_in, trans ? 2 * Fp : Dp, dtype, dx, lddx, c.st));
  // the weights' gradients; of padded operands through a padded copy
  Layer out;
  if (dw_in) {
    void* q = w_ok ? dw_in : c.take(2 * Fp * Dp, we);
    PH_TRY(product(1, 0, w_ok ? 2 * F : 2 * Fp, w_ok ? D : Dp, M, dtype, dab, 2 * Fp, x, ldx, dw_dtype, q, Dp, c.st));
    if (!w_ok) PH_TRY(out.add(q, 2 * F, D, Dp, dw_in, 2 * F, D, false));
  }
  if (dw_out) {
    void* q = w_ok ? dw_out : c.take(Fp * Dp, we);
    PH_TRY(product(1, 0, w_ok ? D : Dp, w_ok ? F : Fp, M, dtype, dy, lddy, h, Fp, dw_dtype, q, Fp, c.st));
    if (!w_ok) PH_TRY(out.add(q, D, F, Fp, dw_out, D, F, false));
  }
  return out.run(dw_dtype, c.st);
}
