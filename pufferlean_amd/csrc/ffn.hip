// Gated feed-forward block y = (act(x Wg^T) * (x Wv^T)) Wo^T and its gradient. With the projections a = x Wg^T and
// v = x Wv^T interleaved in the columns of x w_in^T, h = act(a) v:
//
//   forward   h, p = v act'(a), f = act(a) from one product x w_in^T;  y = h w_out^T
//   backward  dab = (dh p, dh f) interleaved, from one product dh = dy w_out;
//             dw_out = dy^T h;  dw_in = dab^T x;  dx = dab w_in
//
// All on the matrix cores: 6 M D F operations forward and 12 M D F backward, against which the activations' traffic is
// small; the epilogues (glu.hpp) keep the projections and dh from ever being written. bf16 rounds h and dab once each from
// fp32, as operands of bf16 products (up to 64 rows only of those of the weights' gradients); p and f keep 24 bits.
//
// Measured: 65536 x 512 x 1376 bf16 both directions 1234 us, 673 TFLOP/s (357 us h, 298 dab, 350 y and dx, 337 the weights'
// gradients); the products' 592 us at the rate of a large library product are out of reach of their short K of 512.
// 6699 x 203 x 531 fp32 232 us, 56 TFLOP/s: few tiles of padded columns for 256 CUs. 8 rows 12 us, launch and weight latency.
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
// All copies of a call in one launch, a 32 x 32 tile per block. A launch of 2^32 threads or more would start the remainder only,
// so past kLayBlocks tiles a block goes on to its next ones.
constexpr unsigned kLayBlocks = 1u << 20;
template <typename T>
__global__ void __launch_bounds__(256) k_lay(Lays ls) {
  __shared__ T tile[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  for (unsigned at = blockIdx.x; at < ls.blocks; at += gridDim.x) {
    int w = 0;
    while (w + 1 < ls.n && at >= ls.l[w + 1].first) w++;
    const Lay& j = ls.l[w];
    const T* src = (const T*)j.src;
    T* dst = (T*)j.dst;
    const long nc = (j.cols_p + 31) / 32, id = at - j.first, r0 = id / nc * 32, c0 = id % nc * 32;
    if (j.trans) __syncthreads();  // the tile before has been read
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
    if (!j.trans) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      const long c = c0 + y + i, r = r0 + x;
      if (r < j.rows_p && c < j.cols_p) dst[c * j.rows_p + r] = tile[x][y + i];
    }
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
    const unsigned blocks = ls.blocks < kLayBlocks ? ls.blocks : kLayBlocks;
    if (dtype == PH_BF16) k_lay<uint16_t><<<blocks, 256, 0, st>>>(ls);
    else k_lay<float><<<blocks, 256, 0, st>>>(ls);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
};

// ---- few rows --------------------------------------------------------------------------------------------
// Up to 64 rows are bound by the weights' bytes and by latency, so the weights go from memory straight into the operand
// registers of 16-wide products (16 weight rows to a wavefront, 16 bytes of one to a lane), with the rows of x as the
// other operand; the block's wavefronts share the reduction and are added through LDS. fp32 takes four products of
// 16x16x4 for the four values of a lane: the same k of both operands, in an order of its own. What the first product leaves for
// the second is a few KB, so of bf16 blocks it stays fp32 and enters as two bf16 halves, 16 bits: y and dx are rounded once.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
constexpr int kFewRows = 64;

template <typename T> struct Few;
template <> struct Few<uint16_t> {
  static constexpr int kPer = 8;  // k values of a lane
  typedef bf16x8_t Frag;
  static __device__ __forceinline__ Frag load(const uint16_t* row, long k, long K) {
    const uint4 v = k < K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0u, 0u, 0u, 0u);
    return __builtin_bit_cast(bf16x8_t, v);
  }
  static __device__ __forceinline__ f32x4_t mma(Frag a, Frag b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // fp32 values as the sum of two of bf16: the upper half (cut off, so that no finite value becomes infinite), and what is left
  // of it, rounded; nothing is left of an infinity.
  struct Halves {
    Frag hi, lo;
  };
  static __device__ __forceinline__ Halves load(const float* row, long k, long K) {
    f32x4_t v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (k < K) {
      v[0] = *reinterpret_cast<const f32x4_t*>(row + k);
      v[1] = *reinterpret_cast<const f32x4_t*>(row + k + 4);
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float a = v[i / 2][2 * (i % 2)], b = v[i / 2][2 * (i % 2) + 1];
      hi[i] = keep_hi(a, b);
      const float ha = __builtin_bit_cast(float, hi[i] << 16), hb = __builtin_bit_cast(float, hi[i] & 0xffff0000u);
      lo[i] = bf16x2_rne(a == ha ? 0.f : a - ha, b == hb ? 0.f : b - hb);
    }
    return {__builtin_bit_cast(Frag, make_uint4(hi[0], hi[1], hi[2], hi[3])), __builtin_bit_cast(Frag, make_uint4(lo[0], lo[1], lo[2], lo[3]))};
  }
  static __device__ __forceinline__ f32x4_t mma(Frag a, const Halves& b, f32x4_t c) { return mma(a, b.hi, mma(a, b.lo, c)); }
};
template <> struct Few<float> {
  static constexpr int kPer = 4;
  typedef f32x4_t Frag;
  static __device__ __forceinline__ Frag load(const float* row, long k, long K) {
    return k < K ? *reinterpret_cast<const f32x4_t*>(row + k) : f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  static __device__ __forceinline__ f32x4_t mma(Frag a, Frag b, f32x4_t c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ void put(uint16_t* p, float a, float b) { *reinterpret_cast<uint32_t*>(p) = bf16x2_rne(a, b); }
__device__ __forceinline__ void put(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
// Values n .. n + 3, and the pair n, n + 1, of a row of pf (glu.hpp).
__device__ __forceinline__ void keep4(uint16_t* row, long ld, long n, float p0, float f0, float p1, float f1) {
  *reinterpret_cast<uint2*>(row + n) = make_uint2(keep_hi(p0, f0), keep_hi(p1, f1));
  *reinterpret_cast<uint32_t*>(row + ld / 3 * 2 + n / 2) = keep_lo(p0, f0, p1, f1);
}
__device__ __forceinline__ void keep4(float* row, long, long n, float p0, float f0, float p1, float f1) {
  *reinterpret_cast<float4*>(row + n) = make_float4(p0, f0, p1, f1);
}
__device__ __forceinline__ void kept2(const uint16_t* row, long ld, long n, float& p, float& f) {
  const uint32_t hi = *reinterpret_cast<const uint32_t*>(row + n), lo = row[ld / 3 * 2 + n / 2];
  p = kept<0, 0>(hi, lo);
  f = kept<1, 1>(hi, lo);
}
__device__ __forceinline__ void kept2(const float* row, long, long n, float& p, float& f) {
  const float2 u = *reinterpret_cast<const float2*>(row + n);
  p = u.x;
  f = u.y;
}
__device__ __forceinline__ void put1(uint16_t* p, float a) { *p = bf16_rne(a); }
__device__ __forceinline__ void put1(float* p, float a) { *p = a; }

// The product of few rows: out[m][n] = sum_k x[m][k] w[n][k]. kIn: n are the projections, out is h (and pf); kGrad: n are
// units, out is dab, from pf; kPlain: out has N columns. K and the leading dimensions are multiples of 8. X: the type of x. wide
// receives h (dab) in fp32, in out's layout; of the two at least one is there.
enum : int { kIn, kGrad, kPlain };
struct FewArgs {
  const void *x, *w;
  long ldx, ldw, K;
  int M, N, act;
  void* out;
  float* wide;
  long ldo;
  void* pf;
  long ldpf;
};
template <typename T, typename X, int MODE, int MT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) k_few(FewArgs g) {
  __shared__ f32x4_t red[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, w0 = blockIdx.x * 16;
  const T* wr = (const T*)g.w + (long)min(w0 + r, g.N - 1) * g.ldw;  // rows past N and M repeat the last: not stored
  const X* xr[MT];
  f32x4_t acc[MT];
#pragma unroll
  for (int m = 0; m < MT; m++) {
    xr[m] = (const X*)g.x + (long)min(16 * m + r, g.M - 1) * g.ldx;
    acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  constexpr int kPer = Few<T>::kPer, kStep = 4 * kPer;
  const long steps = (g.K + kStep - 1) / kStep, per = (steps + WAVES - 1) / WAVES, beg = wave * per, end = min(steps, beg + per);
  const int ko = kPer * (lane >> 4);
#pragma unroll 4
  for (long s = beg; s < end; s++) {
    const auto a = Few<T>::load(wr, kStep * s + ko, g.K);
#pragma unroll
    for (int m = 0; m < MT; m++) acc[m] = Few<T>::mma(a, Few<T>::load(xr[m], kStep * s + ko, g.K), acc[m]);
  }
#pragma unroll
  for (int m = 0; m < MT; m++) red[wave][m][lane] = acc[m];
  __syncthreads();
  if (wave >= MT) return;
  f32x4_t s = red[0][wave][lane];
  for (int v = 1; v < WAVES; v++) s += red[v][wave][lane];
  // the lane has columns n..n+3 of one row
  const int row = 16 * wave + r, n = w0 + 4 * (lane >> 4);
  if (row >= g.M || n >= g.N) return;
  T* out = g.out ? (T*)g.out + (long)row * g.ldo : nullptr;
  float* wide = MODE != kPlain && g.wide ? g.wide + (long)row * g.ldo : nullptr;
  T* pf = g.pf ? (T*)g.pf + (long)row * g.ldpf : nullptr;
  if constexpr (MODE == kIn) {
    float f0, d0, f1, d1;
    glu_act(g.act, s[0], f0, d0);
    glu_act(g.act, s[2], f1, d1);
    const float h0 = f0 * s[1], h1 = f1 * s[3];
    if (out) put(out + n / 2, h0, h1);
    if (wide) put(wide + n / 2, h0, h1);
    if (pf) keep4(pf, g.ldpf, n, s[1] * d0, f0, s[3] * d1, f1);
  } else if constexpr (MODE == kGrad) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float p, f;
      kept2(pf, g.ldpf, 2 * (n + i), p, f);
      if (out) put(out + 2 * (n + i), s[i] * p, s[i] * f);
      if (wide) put(wide + 2 * (n + i), s[i] * p, s[i] * f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (n + i < g.N) put1(out + n + i, s[i]);
  }
}

template <typename T, typename X, int MODE>
int few_t(const FewArgs& g, hipStream_t st) {
  const unsigned blocks = (unsigned)((g.N + 15) / 16);
  if (g.M <= 16) k_few<T, X, MODE, 1, 8><<<blocks, 512, 0, st>>>(g);
  else if (g.M <= 32) k_few<T, X, MODE, 2, 8><<<blocks, 512, 0, st>>>(g);
  else k_few<T, X, MODE, 4, 8><<<blocks, 512, 0, st>>>(g);
  PH_LAUNCH_CHECK();
  return PH_OK;
}
// x in dtype, of kPlain in fp32.
template <int MODE>
int few(int dtype, const FewArgs& g, hipStream_t st) {
  typedef std::conditional_t<MODE == kPlain, float, uint16_t> X;
  return dtype == PH_BF16 ? few_t<uint16_t, X, MODE>(g, st) : few_t<float, float, MODE>(g, st);
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

// A weight's gradient A^T B over the M rows. A few hundred tiles of 64x64 at most, each a long sum, leave the chip idle or its
// blocks without company: enough splits for six blocks to a CU, of 256 rows at least (fp32 1072x208x6699 90 -> 57 us,
// 208x536x6699 45 -> 35, 2752x512x4096 258 -> 157). bf16 keeps gemm()'s own choice (3592 rows, 2208x384 and 384x1104: 54 us, 66
// this way).
int weight_grad(size_t rows, size_t cols, size_t M, int dtype, const void* A, size_t lda, const void* B, size_t ldb, int c_dtype,
                void* C, hipStream_t st) {
  PhGemmDesc d{};
  d.trans_a = 1; d.M = (int)rows; d.N = (int)cols; d.K = (int)M;
  d.a_dtype = d.b_dtype = dtype; d.A = A; d.lda = (long)lda; d.B = B; d.ldb = (long)ldb;
  d.c_dtype = c_dtype; d.C = C; d.ldc = (long)cols;
  d.math = dtype == PH_BF16 ? PH_MATH_BF16 : PH_MATH_F32;
  const long tiles = (long)((rows + 63) / 64) * (long)((cols + 63) / 64);
  if (dtype == PH_F32 && M >= 512 && tiles < 768) {
    const long want = (1536 + tiles - 1) / tiles, most = (long)M / 256;
    d.splits = (int)(want < most ? want : most);
    d.small_tiles = 1;
  }
  return gemm(d, st);
}

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
  // the second product's operand where h is not it: few rows of bf16 units take it in fp32
  const bool few_rows = M <= (size_t)kFewRows, wide = few_rows && dtype == PH_BF16;
  if (wide) c.want(M * Fp, 4);
  else if (!h) c.want(M * Fp, c.e);
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
  float* hw = wide ? (float*)c.take(M * Fp, 4) : nullptr;
  if (!h && !wide) h = c.take(M * Fp, c.e);
  if (few_rows) {
    FewArgs g{};
    g.x = x; g.ldx = (long)ldx; g.w = w_in; g.ldw = g.K = (long)Dp; g.M = (int)M; g.N = (int)(2 * Fp); g.act = act;
    g.out = h; g.wide = hw; g.ldo = (long)Fp; g.pf = pf; g.ldpf = keep_pitch(dtype, (long)Fp);
    PH_TRY(few<kIn>(dtype, g, c.st));
    FewArgs o{};
    o.x = wide ? hw : h; o.ldx = (long)Fp; o.w = w_out; o.ldw = o.K = (long)Fp; o.M = (int)M; o.N = (int)D; o.out = y; o.ldo = (long)ldy;
    return few<kPlain>(dtype, o, c.st);
  }
  GluProduct g{};
  g.dtype = dtype; g.act = act; g.M = (int)M; g.N = (int)(2 * Fp); g.K = (int)Dp;
  g.A = x; g.lda = (long)ldx; g.B = w_in; g.ldb = (long)Dp; g.h = h; g.ldh = (long)Fp; g.pf = pf; g.ldpf = keep_pitch(dtype, (long)Fp);
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
  // are faster by more than the copies take, and the kernel of few rows has no other form. In between the products
  // take the weights as they are (or padded).
  const bool few_rows = M <= (size_t)kFewRows, trans = M >= kTransposeRows || few_rows;
  const bool wide = few_rows && dtype == PH_BF16;  // dx from fp32 gradients of the projections
  const bool wo_ok = !trans && c.whole(w_out, F, F, Fp) && D == Dp, wi_ok = !trans && c.whole(w_in, D, D, Dp) && F == Fp;
  const bool need_dab = dx || dw_in;
  if (!x_ok && dw_in) c.want(M * Dp, c.e);
  if (!dy_ok) c.want(M * Dp, c.e);
  if (need_dab) {
    if (!wo_ok) c.want(Fp * Dp, c.e);
    if (!wi_ok && dx) c.want(2 * Fp * Dp, c.e);
    if (!wide || dw_in) c.want(M * 2 * Fp, c.e);
    if (wide && dx) c.want(M * 2 * Fp, 4);
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
  float* dabw = nullptr;
  if (need_dab) {
    if (!wo_ok) PH_TRY(laid(w_out, D, F, F, Dp, Fp, trans));
    if (!wi_ok && dx) PH_TRY(laid(w_in, 2 * F, D, D, 2 * Fp, Dp, trans));
    if (!wide || dw_in) dab = c.take(M * 2 * Fp, c.e);
    if (wide && dx) dabw = (float*)c.take(M * 2 * Fp, 4);
  }
  PH_TRY(lay.run(dtype, c.st));
  if (need_dab && few_rows) {
    FewArgs g{};
    g.x = dy; g.ldx = (long)lddy; g.w = w_out; g.ldw = g.K = (long)Dp; g.M = (int)M; g.N = (int)Fp; g.out = dab; g.wide = dabw; g.ldo = (long)(2 * Fp);
    g.pf = const_cast<void*>(pf); g.ldpf = keep_pitch(dtype, (long)Fp);
    PH_TRY(few<kGrad>(dtype, g, c.st));
  } else if (need_dab) {
    GluProduct g{};
    g.grad = 1; g.dtype = dtype; g.act = act; g.M = (int)M; g.N = (int)Fp; g.K = (int)Dp; g.b_kn = !trans;
    g.A = dy; g.lda = (long)lddy; g.B = w_out; g.ldb = (long)(trans ? Dp : Fp);
    g.pf = const_cast<void*>(pf); g.ldpf = keep_pitch(dtype, (long)Fp); g.dab = dab; g.lddab = (long)(2 * Fp);
    PH_TRY(glu_product(g, c.st));
  }
  // the weights' gradients; of padded operands through a padded copy
  Layer out;
  if (dw_in) {
    void* q = w_ok ? dw_in : c.take(2 * Fp * Dp, we);
    PH_TRY(weight_grad(w_ok ? 2 * F : 2 * Fp, w_ok ? D : Dp, M, dtype, dab, 2 * Fp, x, ldx, dw_dtype, q, c.st));
    if (!w_ok) PH_TRY(out.add(q, 2 * F, D, Dp, dw_in, 2 * F, D, false));
  }
  if (dw_out) {
    void* q = w_ok ? dw_out : c.take(Fp * Dp, we);
    PH_TRY(weight_grad(w_ok ? D : Dp, w_ok ? F : Fp, M, dtype, dy, lddy, h, Fp, dw_dtype, q, c.st));
    if (!w_ok) PH_TRY(out.add(q, D, F, Fp, dw_out, D, F, false));
  }
  // dx last: it may be written over x or dy
  if (dx && few_rows) {
    FewArgs g{};
    g.x = wide ? dabw : dab; g.ldx = (long)(2 * Fp); g.w = w_in; g.ldw = g.K = (long)(2 * Fp); g.M = (int)M; g.N = (int)D; g.out = dx; g.ldo = (long)lddx;
    PH_TRY(few<kPlain>(dtype, g, c.st));
  } else if (dx) PH_TRY(product(0, trans, M, D, 2 * Fp, dtype, dab, 2 * Fp, w_in, trans ? 2 * Fp : Dp, dtype, dx, lddx, c.st));
  return out.run(dw_dtype, c.st);
}
