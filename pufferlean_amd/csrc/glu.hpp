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

// Product with the gated unit in its epilogue, C[M x N] = A[M x K] B[N x K]^T (b_kn: B stored [K][N]), all of one type; N, K and the leading
// dimensions are multiples of 8 and the pointers 16-byte aligned.
//   grad 0: columns 2j, 2j+1 are unit j's gate and value projections a, v. h[row][j] = act(a) v, and (pf not NULL)
//           pf[row][2j..] = v act'(a), act(a): what the gradient multiplies dh with, rounded once.
//   grad 1: the columns are dh; dab[row][2j..] = dh pf[row][2j..], the projections' gradients.
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
