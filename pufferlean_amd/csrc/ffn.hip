// Gated feed-forward block y = (act(x Wg^T) * (x Wv^T)) Wo^T and its gradient. With the projections a = x Wg^T and
// v = x Wv^T interleaved in the columns of ab = x w_in^T, h = act(a) v:
//
//   forward   ab = x w_in^T, h;  y = h w_out^T
//   backward  dh = dy w_out;  da = dh v act'(a), dv = dh act(a) (interleaved in dab);
//             dw_out = dy^T h;  dw_in = dab^T x;  dx = dab w_in
//
// Three products each way (a product twice as wide counts twice), all on the matrix cores.
#include "common.hpp"
#include "kernels.hpp"

namespace ph {
namespace {

__device__ __forceinline__ float ldf(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ void stf(uint16_t* p, float v) { *p = bf16_rne(v); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }

// The activation and its derivative.
__device__ __forceinline__ void act_of(int act, float a, float& f, float& df) {
  if (act == PH_ACT_SILU) {
    const float s = sigm(a);
    f = a * s;
    df = s * fmaf(a, 1.f - s, 1.f);
  } else {
    const float p = 0.5f * erfcf(a * -0.70710678118654752f);
    f = a * p;
    df = fmaf(a * 0.39894228040143268f, __expf(-0.5f * a * a), p);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_glu_fwd(const T* __restrict__ ab, long ldab, T* __restrict__ h, long ldh, long M, int F,
                                                 int act) {
  const long n = M * F;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / F, j = i % F;
    float f, df;
    act_of(act, ldf(ab + r * ldab + 2 * j), f, df);
    stf(h + r * ldh + j, f * ldf(ab + r * ldab + 2 * j + 1));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_glu_bwd(const T* __restrict__ ab, long ldab, const float* __restrict__ dh, long lddh,
                                                 T* __restrict__ dab, long lddab, long M, int F, int act) {
  const long n = M * F;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / F, j = i % F;
    float f, df;
    const float g = dh[r * lddh + j], v = ldf(ab + r * ldab + 2 * j + 1);
    act_of(act, ldf(ab + r * ldab + 2 * j), f, df);
    stf(dab + r * lddab + 2 * j, g * v * df);
    stf(dab + r * lddab + 2 * j + 1, g * f);
  }
}

unsigned elementwise_blocks(size_t n) {
  const unsigned b = ceil_div(n, 256);
  return b < 16384 ? b : 16384;
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

size_t pitch(size_t cols) { return (cols + 7) / 8 * 8; }

int check(const char* who, int dtype, int act, size_t M, size_t D, size_t F) {
  PH_REQUIRE(dtype == PH_F32 || dtype == PH_BF16, "%s: dtype must be F32 or BF16", who);
  PH_REQUIRE(act == PH_ACT_SILU || act == PH_ACT_GELU, "%s: unknown activation %d", who, act);
  PH_REQUIRE(D >= 1 && F >= 1 && D <= (1u << 20) && F <= (1u << 20) && M <= (1u << 30), "%s: M = %zu, D = %zu, F = %zu out of range",
             who, M, D, F);
  return PH_OK;
}

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" size_t ph_ffn_pitch(size_t columns) { return pitch(columns); }

extern "C" int ph_ffn(int dtype, int act, size_t M, size_t D, size_t F, const void* x, size_t ldx, const void* w_in,
                      const void* w_out, void* ab, void* h, void* y, size_t ldy, void* stream) {
  PH_TRY(check("ffn", dtype, act, M, D, F));
  PH_REQUIRE(ldx >= D && ldy >= D, "ffn: row strides %zu, %zu below %zu columns", ldx, ldy, D);
  if (M == 0) return PH_OK;
  PH_REQUIRE(x && w_in && w_out && y, "ffn: x, w_in, w_out or y missing");
  PH_REQUIRE(!ab == !h, "ffn: ab and h are kept together");
  hipStream_t st = as_stream(stream);
  const size_t e = dtype == PH_BF16 ? 2 : 4, pab = pitch(2 * F), ph_ = pitch(F);
  if (!ab) {
    uint8_t* ws = (uint8_t*)scratch(kSlotFfn, M * (pab + ph_) * e);
    if (!ws) return PH_ERR_NOMEM;
    ab = ws;
    h = ws + M * pab * e;
  }
  PH_TRY(product(0, 1, M, 2 * F, D, dtype, x, ldx, w_in, D, dtype, ab, pab, st));
  if (dtype == PH_BF16)
    k_glu_fwd<uint16_t><<<elementwise_blocks(M * F), 256, 0, st>>>((const uint16_t*)ab, pab, (uint16_t*)h, ph_, M, (int)F, act);
  else k_glu_fwd<float><<<elementwise_blocks(M * F), 256, 0, st>>>((const float*)ab, pab, (float*)h, ph_, M, (int)F, act);
  PH_LAUNCH_CHECK();
  return product(0, 1, M, D, F, dtype, h, ph_, w_out, F, dtype, y, ldy, st);
}

extern "C" int ph_ffn_grad(int dtype, int act, size_t M, size_t D, size_t F, const void* x, size_t ldx, const void* w_in,
                           const void* w_out, const void* ab, const void* h, const void* dy, size_t lddy, void* dx,
                           size_t lddx, int dw_dtype, void* dw_in, void* dw_out, void* stream) {
  PH_TRY(check("ffn_grad", dtype, act, M, D, F));
  PH_REQUIRE(dw_dtype == dtype || dw_dtype == PH_F32, "ffn_grad: the weights' gradients are of dtype or F32");
  PH_REQUIRE(ldx >= D && lddy >= D && (!dx || lddx >= D), "ffn_grad: a row stride is below %zu columns", D);
  PH_REQUIRE(M == 0 || (x && w_in && w_out && ab && h && dy), "ffn_grad: an input is missing");
  hipStream_t st = as_stream(stream);
  const size_t e = dtype == PH_BF16 ? 2 : 4, pab = pitch(2 * F), ph_ = pitch(F);
  if (M > 0 && (dx || dw_in)) {
    uint8_t* ws = (uint8_t*)scratch(kSlotFfn, M * (pab * e + ph_ * 4));
    if (!ws) return PH_ERR_NOMEM;
    void* dab = ws;
    float* dh = (float*)(ws + M * pab * e);
    PH_TRY(product(0, 0, M, F, D, dtype, dy, lddy, w_out, F, PH_F32, dh, ph_, st));
    if (dtype == PH_BF16)
      k_glu_bwd<uint16_t><<<elementwise_blocks(M * F), 256, 0, st>>>((const uint16_t*)ab, pab, dh, ph_, (uint16_t*)dab, pab, M, (int)F, act);
    else k_glu_bwd<float><<<elementwise_blocks(M * F), 256, 0, st>>>((const float*)ab, pab, dh, ph_, (float*)dab, pab, M, (int)F, act);
    PH_LAUNCH_CHECK();
    if (dx) PH_TRY(product(0, 0, M, D, 2 * F, dtype, dab, pab, w_in, D, dtype, dx, lddx, st));
    if (dw_in) PH_TRY(product(1, 0, 2 * F, D, M, dtype, dab, pab, x, ldx, dw_dtype, dw_in, D, st));
  } else if (dw_in) {
    PH_TRY(product(1, 0, 2 * F, D, 0, dtype, nullptr, pab, nullptr, D, dw_dtype, dw_in, D, st));
  }
  if (dw_out) PH_TRY(product(1, 0, D, F, M, dtype, dy, lddy, h, ph_, dw_dtype, dw_out, F, st));
  return PH_OK;
}
