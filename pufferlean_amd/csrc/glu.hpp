// Activations of the gated feed-forward units, shared by the product whose epilogue applies them and by the kernels of few
// rows.
#pragma once
#include "common.hpp"

namespace ph {

// act(a) and its derivative: a sigma(a), or a Phi(a) with the normal distribution function Phi.
__device__ __forceinline__ void glu_act(int act, float a, float& f, float& df) {
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

// What the gradient multiplies dh with: a unit's pair p = v act'(a), f = act(a), rows of them, pf. Their roundings would add to
// those of the products' operands (a bf16 pair makes dx and dw_in 1.7 times as far from their exact values as one rounding of
// the result; this way 1.4 times), so of bf16 units a pair has the first 24 bits of its fp32 values, 16 of mantissa, cut off: an
// error of 2^-15 at most, where a bf16 operand's rounding costs up to 2^-8. The upper 16 bits of a row's 2F values come first,
// then the next 8 of each. A row is keep_pitch values of the units' type.
inline long keep_pitch(int dtype, long F) { return (dtype == PH_BF16 ? 3 : 2) * F; }
// The upper halves of two fp32 values, and the bytes behind those of four.
__device__ __forceinline__ uint32_t keep_hi(float a, float b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302);
}
__device__ __forceinline__ uint32_t keep_lo(float a, float b, float c, float d) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x0c0c0501) |
         __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, d), __builtin_bit_cast(uint32_t, c), 0x05010c0c);
}
// Value j of the two in hi, with byte k of lo.
template <int J, int K> __device__ __forceinline__ float kept(uint32_t hi, uint32_t lo) {
  return __builtin_bit_cast(float, __builtin_amdgcn_perm(hi, lo, (J ? 0x07060000u : 0x05040000u) | K << 8 | 0x0cu));
}

// Product with the gated unit in its epilogue, C[M x N] = A[M x K] B[N x K]^T (b_kn: B stored [K][N]), all of one type; N, K and the leading
// dimensions are multiples of 8 and the pointers 16-byte aligned.
//   grad 0: columns 2j, 2j+1 are unit j's gate and value projections a, v. h[row][j] = act(a) v, and (pf not NULL)
//           pf[row] as above.
//   grad 1: the columns are dh; dab[row][2j..] = dh p, dh f, the projections' gradients.
struct GluProduct {
  int grad, dtype, act, M, N, K, b_kn;
  const void* A;
  long lda;
  const void* B;
  long ldb;
  void* h;
  long ldh;
  void* pf;
  long ldpf;
  void* dab;
  long lddab;
};
int glu_product(const GluProduct& p, hipStream_t st);

}  // namespace ph
