// Selective state-space scan with its short causal convolution, for sequences (forward and gradient) and single
// tokens. Per sequence b, channel c and step t, time-major:
//
//   u_t  = silu(conv_b + sum_k conv_w[k] x_{t-K+1+k})     (u_t = x_t without a convolution)
//   d_t  = softplus(delta_t + dt_bias)
//   h_t  = exp(d_t A) h_{t-1} + d_t u_t B_t               (N states per channel; B_t, C_t shared by a group's channels)
//   y_t  = (<h_t, C_t> + D u_t) [ * z_t sigma(z_t) ]
//
// A step after the end of an episode starts from a cleared state and an empty convolution window.
//
// Layout. A lane owns one channel and all its N states in registers, a wavefront 64 channels of one sequence,
// so the only values that cross lanes are B_t and C_t, which every lane of the block reads from LDS as broadcasts
// (staged there kSteps steps at a time, converted once). The state stays in fp32 throughout and is never
// written per step; what a step costs is vector arithmetic: per state one exponential (a quarter-rate
// instruction, 16 cycles of a wavefront), the decay's argument, the input, the update and the output (4 cycles
// each), 32 cycles in all against 8 bytes of memory per channel and step.
//
// Long sequences of few channels do not fill the chip with one wavefront per 64 channels, so time is cut into
// chunks: a first launch runs every chunk from a zero state and keeps its end state and the sum of d_t (the
// chunk's decay is exp(A sum d)), a second joins the chunks' start states in order, and the third runs the
// chunks again from those.
#include "common.hpp"
#include "kernels.hpp"

#include <cmath>

namespace ph {
namespace {

constexpr int kSteps = 8;  // steps of a batch: staged, prefetched and (N <= 16) kept together
constexpr int kTaps = 4;   // most taps of the convolution; fewer are padded with zero taps in front
constexpr int kMaxStates = 64;
constexpr float kLog2e = 1.4426950408889634f;

// Steps between two kept states of the training forward: the backward holds that many steps' states in registers.
constexpr int keep_steps(int ns) { return ns <= 16 ? 8 : (ns <= 32 ? 4 : 2); }
// States of a lane's registers: the least of these that holds N.
constexpr int states_of(long N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

// Wavefronts of a block of the gradient: two to a SIMD where the states fit 256 registers, else one.
constexpr int bwd_waves(int ns) { return ns <= 16 ? 8 : 4; }

struct Args {
  long T, B, C, N, per, K;  // per: channels of a group
  const void *x, *z, *delta, *Bm, *Cm;
  long x_t, x_b, z_t, z_b, d_t, d_b, bm_t, bm_b, cm_t, cm_b;
  const float *A, *D, *dt_bias, *conv_w, *conv_b;
  const float *done, *first, *h0, *win0;
  void* y;
  long y_t, y_b;
  float *h_out, *keep;
  long chunk, chunks;   // steps of a chunk (a multiple of kSteps), their number
  float *hloc, *dsum;   // [chunks][B][C][N] end (then start) states, [chunks][B][C] sums of d (-1: cleared inside)
  int blocks_c;         // channel blocks of a group
};

__device__ __forceinline__ float ldf(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ void stf(uint16_t* p, float v) { *p = bf16_rne(v); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }

__device__ __forceinline__ float ex2(float v) { return __builtin_amdgcn_exp2f(v); }
// softplus without cancellation: with w = 1 + e rounded, log(w) e / (w - 1) is log(1 + e) to a few ulp for every e.
__device__ __forceinline__ float softplus(float v) {
  const float e = __expf(-fabsf(v)), w = 1.f + e;
  const float l = w == 1.f ? e : __logf(w) * (e / (w - 1.f));
  return fmaxf(v, 0.f) + l;
}

// The convolution's rolling window: the three inputs before the current one (those past K - 1 steps back stay 0).
struct Conv {
  float w[kTaps], bias;
  float p[kTaps - 1];
  int K;
  __device__ __forceinline__ void init(const Args& a, long c) {
    K = (int)a.K;
#pragma unroll
    for (int i = 0; i < kTaps; i++) {
      const int k = i - (kTaps - K);
      w[i] = K > 0 && k >= 0 ? a.conv_w[c * K + k] : 0.f;
    }
    bias = K > 0 && a.conv_b ? a.conv_b[c] : 0.f;
    clear();
  }
  __device__ __forceinline__ void clear() { p[0] = p[1] = p[2] = 0.f; }
  __device__ __forceinline__ float pre(float x) const {
    return fmaf(w[3], x, fmaf(w[2], p[2], fmaf(w[1], p[1], fmaf(w[0], p[0], bias))));
  }
  __device__ __forceinline__ void push(float x) {
    p[0] = K >= 4 ? p[1] : 0.f;
    p[1] = K >= 3 ? p[2] : 0.f;
    p[2] = K >= 2 ? x : 0.f;
  }
};
__device__ __forceinline__ float silu(float v) { return v * sigm(v); }

// Whether step t of sequence b starts an episode.
__device__ __forceinline__ bool starts(const Args& a, long t, long b) {
  if (t > 0) return a.done && a.done[(t - 1) * a.B + b] != 0.f;
  return a.first && a.first[b] != 0.f;
}

// The window as it stands before step t0: the last K - 1 inputs, of the sequence or of the carried window.
template <typename T>
__device__ __forceinline__ void conv_seek(Conv& cv, const Args& a, long t0, long b, long c) {
  if (cv.K < 2) return;
  for (long t = t0 - (cv.K - 1); t < t0; t++) {
    float v;
    if (t < 0) v = a.win0 ? a.win0[(b * (cv.K - 1) + cv.K - 1 + t) * a.C + c] : 0.f;
    else {
      if (starts(a, t, b)) cv.clear();
      v = ldf((const T*)a.x + t * a.x_t + b * a.x_b + c);
    }
    cv.push(v);
  }
}

struct Place {
  long b, s, c, c0;  // sequence, chunk, this lane's channel (clamped into the group), the group's first channel
  int g;
  bool in;           // whether the lane has a channel
};
__device__ __forceinline__ Place place(const Args& a, long id) {
  Place p;
  const int cb = (int)(id % a.blocks_c);
  id /= a.blocks_c;
  const long G = a.C / a.per;
  p.g = (int)(id % G);
  id /= G;
  p.b = id % a.B;
  p.s = id / a.B;
  const long lc = (long)cb * blockDim.x + threadIdx.x;
  p.in = lc < a.per;
  p.c0 = (long)p.g * a.per;
  p.c = p.c0 + (p.in ? lc : a.per - 1);
  return p;
}

// B and C of kSteps steps from t0 as fp32 in LDS, [step][2][NS], zero past N and past the sequence's end.
template <typename T, int NS>
__device__ __forceinline__ void stage_bc(float* s, const Args& a, long t0, long tend, long b, int g) {
  const int tot = kSteps * 2 * NS;
  for (int e = threadIdx.x; e < tot; e += blockDim.x) {
    const int n = e % NS, which = (e / NS) & 1;
    const long t = t0 + e / (2 * NS);
    float v = 0.f;
    if (n < a.N && t < tend) {
      const long col = g * a.N + n;
      v = which ? ldf((const T*)a.Cm + t * a.cm_t + b * a.cm_b + col)
                : ldf((const T*)a.Bm + t * a.bm_t + b * a.bm_b + col);
    }
    s[e] = v;
  }
}

template <int NS>
__device__ __forceinline__ void load_state(float (&h)[NS], const float* p, long N) {
#pragma unroll
  for (int n = 0; n < NS; n++) h[n] = n < N ? p[n] : 0.f;
}
template <int NS>
__device__ __forceinline__ void store_state(float* p, const float (&h)[NS], long N) {
#pragma unroll
  for (int n = 0; n < NS; n++)
    if (n < N) p[n] = h[n];
}

// One chunk of one sequence. LOCAL: from a zero state, keeping only the end state and the decay's exponent.
template <typename T, int NS, bool LOCAL>
__global__ void __launch_bounds__(256) k_ssm_fwd(Args a) {
  __shared__ __attribute__((aligned(16))) float sbc[kSteps * 2 * NS];
  const Place pl = place(a, blockIdx.x);
  const long b = pl.b, c = pl.c;
  const long tbeg = pl.s * a.chunk, tend = min(a.T, tbeg + a.chunk);
  Conv cv;
  cv.init(a, c);
  conv_seek<T>(cv, a, tbeg, b, c);
  float A2[NS], h[NS];
#pragma unroll
  for (int n = 0; n < NS; n++) A2[n] = n < a.N ? a.A[c * a.N + n] * kLog2e : 0.f;
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
  const long hoff = (b * a.C + c) * a.N;
  if (LOCAL || (a.chunks == 1 && !a.h0)) {
#pragma unroll
    for (int n = 0; n < NS; n++) h[n] = 0.f;
  } else {
    load_state<NS>(h, a.chunks > 1 ? a.hloc + pl.s * a.B * a.C * a.N + hoff : a.h0 + hoff, a.N);
  }
  float dsum = 0.f;
  bool cleared = false;
  const T* xp = (const T*)a.x + b * a.x_b + c;
  const T* dp = (const T*)a.delta + b * a.d_b + c;
  const T* zp = (const T*)a.z + (a.z ? b * a.z_b + c : 0);
  T* yp = (T*)a.y + b * a.y_b + c;
  for (long t0 = tbeg; t0 < tend; t0 += kSteps) {
    float rx[kSteps], rd[kSteps], rz[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const long t = min(t0 + i, tend - 1);
      rx[i] = ldf(xp + t * a.x_t);
      rd[i] = ldf(dp + t * a.d_t);
      rz[i] = !LOCAL && a.z ? ldf(zp + t * a.z_t) : 0.f;
    }
    __syncthreads();
    stage_bc<T, NS>(sbc, a, t0, tend, b, pl.g);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const long t = t0 + i;
      if (t >= tend) break;
      if (!LOCAL && a.keep && i % keep_steps(NS) == 0 && pl.in)
        store_state<NS>(a.keep + (t / keep_steps(NS)) * a.B * a.C * a.N + hoff, h, a.N);
      if (starts(a, t, b)) {
        cv.clear();
        cleared = true;
#pragma unroll
        for (int n = 0; n < NS; n++) h[n] = 0.f;
      }
      const float x = rx[i];
      const float u = cv.K ? silu(cv.pre(x)) : x;
      cv.push(x);
      const float d = softplus(rd[i] + bias), du = d * u;
      dsum += d;
      float o = Dc * u;
#pragma unroll
      for (int n = 0; n < NS; n++) {
        h[n] = fmaf(ex2(d * A2[n]), h[n], du * sbc[i * 2 * NS + n]);
        if (!LOCAL) o = fmaf(h[n], sbc[(i * 2 + 1) * NS + n], o);
      }
      if (!LOCAL && pl.in) stf(yp + t * a.y_t, a.z ? o * silu(rz[i]) : o);
    }
  }
  if (!pl.in) return;
  if (LOCAL) {
    store_state<NS>(a.hloc + pl.s * a.B * a.C * a.N + hoff, h, a.N);
    a.dsum[(pl.s * a.B + b) * a.C + c] = cleared ? -1.f : dsum;
  } else if (tend == a.T && a.h_out) {
    store_state<NS>(a.h_out + hoff, h, a.N);
  }
}

// Joins the chunks in order: hloc[s] becomes the state before chunk s. One thread per state.
__global__ void __launch_bounds__(256) k_ssm_join(Args a) {
  const long BCN = a.B * a.C * a.N, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= BCN) return;
  const long bc = i / a.N, c = bc % a.C, n = i % a.N;
  const float A2 = a.A[c * a.N + n] * kLog2e;
  float run = a.h0 ? a.h0[i] : 0.f;
  for (long s = 0; s < a.chunks; s++) {
    const float loc = a.hloc[s * BCN + i], d = a.dsum[s * a.B * a.C + bc];
    a.hloc[s * BCN + i] = run;
    run = d < 0.f ? loc : fmaf(ex2(A2 * d), run, loc);
  }
}

// The window after the last step: its K - 1 inputs, zero where an episode started after them. A launch of its own, so
// that it may overwrite the window that the scan read.
template <typename T>
__global__ void __launch_bounds__(256) k_ssm_window(Args a, float* win) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * a.C) return;
  const long b = i / a.C, c = i % a.C;
  Conv cv;
  cv.init(a, c);
  conv_seek<T>(cv, a, a.T, b, c);
  for (int k = 0; k < cv.K - 1; k++) win[(b * (cv.K - 1) + k) * a.C + c] = cv.p[kTaps - cv.K + k];
}

// ---- single tokens -------------------------------------------------------------------------------------
// One step of every sequence, the state updated in place: bound by the state's 8 bytes per element. Four lanes'
// worth of a channel: each lane holds four consecutive states (one 16-byte access each way), LPC lanes a channel.
template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(256) k_ssm_step(Args a, float* __restrict__ hs, float* __restrict__ win) {
  const long nb = (a.C + 256 / LPC - 1) / (256 / LPC), b = blockIdx.x / nb;
  const long cc = (blockIdx.x % nb) * (256 / LPC) + threadIdx.x / LPC;
  const bool in = cc < a.C;  // the lanes of a channel agree; the shuffles stay inside them
  const long c = in ? cc : a.C - 1;
  const int n0 = (threadIdx.x % LPC) * 4, N = (int)a.N;
  const bool clear = a.first && a.first[b] != 0.f;
  float* hp = hs + (b * a.C + c) * N + n0;
  float h[4], Av[4], Bv[4], Cv[4];
  if constexpr (VEC) {
    const float4 hv = *reinterpret_cast<const float4*>(hp), av = *reinterpret_cast<const float4*>(a.A + c * N + n0);
    h[0] = hv.x; h[1] = hv.y; h[2] = hv.z; h[3] = hv.w;
    Av[0] = av.x; Av[1] = av.y; Av[2] = av.z; Av[3] = av.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const bool ok = n0 + i < N;
      h[i] = ok ? hp[i] : 0.f;
      Av[i] = ok ? a.A[c * N + n0 + i] : 0.f;
    }
  }
  const long g = c / a.per;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const bool ok = n0 + i < N;
    Bv[i] = ok ? ldf((const T*)a.Bm + b * a.bm_b + g * N + n0 + i) : 0.f;
    Cv[i] = ok ? ldf((const T*)a.Cm + b * a.cm_b + g * N + n0 + i) : 0.f;
  }
  const float x = ldf((const T*)a.x + b * a.x_b + c);
  const int K = (int)a.K;
  float u = x;
  if (K) {
    float s = a.conv_b ? a.conv_b[c] : 0.f;
    float p[kTaps - 1] = {};
    for (int k = 0; k < K - 1; k++) {
      p[k] = clear ? 0.f : win[(b * (K - 1) + k) * a.C + c];
      s = fmaf(a.conv_w[c * K + k], p[k], s);
    }
    s = fmaf(a.conv_w[c * K + K - 1], x, s);
    u = silu(s);
    // one lane of the channel moves the window on; its wavefront's loads of it are done (they fed s)
    if (in && n0 == 0)
      for (int k = 0; k < K - 1; k++) win[(b * (K - 1) + k) * a.C + c] = k + 1 < K - 1 ? p[k + 1] : x;
  }
  const float d = softplus(ldf((const T*)a.delta + b * a.d_b + c) + (a.dt_bias ? a.dt_bias[c] : 0.f)), du = d * u;
  float o = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    h[i] = fmaf(ex2(d * (Av[i] * kLog2e)), clear ? 0.f : h[i], du * Bv[i]);
    o = fmaf(h[i], Cv[i], o);
  }
  if (in) {
    if constexpr (VEC) {
      *reinterpret_cast<float4*>(hp) = make_float4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (n0 + i < N) hp[i] = h[i];
    }
  }
#pragma unroll
  for (int m = 1; m < LPC; m <<= 1) o += __shfl_xor(o, m);
  if (in && n0 == 0) {
    o = fmaf(a.D ? a.D[c] : 0.f, u, o);
    if (a.z) o *= silu(ldf((const T*)a.z + b * a.z_b + c));
    stf((T*)a.y + b * a.y_b + c, o);
  }
}

// ---- gradient ------------------------------------------------------------------------------------------
struct GradArgs {
  const void* dy;
  long dy_t, dy_b;
  void *dx, *dz, *ddelta, *dB, *dC;
  long dx_t, dx_b, dz_t, dz_b, dd_t, dd_b, db_t, db_b, dc_t, dc_b;
  const float* keep;
  float* carry;   // [chunks][B][C][N]: each chunk's own adjoint at its start, then the one coming in at its end
  float* bc;      // [blocks_c][T][B][G][2][N] sums of dB, dC over a block's channels
  float* par;     // [rows][C][P] sums of the parameters' gradients over a block's work, P = N + K + 3
  float* halo;    // [chunks][B][K-1][C]: what a chunk adds to dx of the K - 1 steps before it
  long rows;      // blocks that share a channel block's work
  int P;
};

// Sum of NV values over the 64 lanes, each value's result left in lanes of its own. Two values at a time are folded
// by swapping wavefront halves, then rows of 16 lanes, then by lane permutations inside a row, so NV values take
// about 2 NV instructions instead of 6 NV.
template <int CTL> __device__ __forceinline__ float dpp_mov(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTL, 0xF, 0xF, true));
}
// Two registers with one's upper and the other's lower wavefront half (or odd and even rows of 16 lanes) exchanged, two pairs
// at a time: their sum then holds the first value's total in one half and the second's in the other. As asm: the
// compiler's builtins return the first register for both. The exchange may not read a register in the two wait
// states after vector arithmetic wrote it, hence the s_nop.
__device__ __forceinline__ void swap32(float& a0, float& b0, float& a1, float& b1) {
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_permlane32_swap_b32 %2, %3" : "+v"(a0), "+v"(b0), "+v"(a1), "+v"(b1));
}
__device__ __forceinline__ void swap16(float& a0, float& b0, float& a1, float& b1) {
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3" : "+v"(a0), "+v"(b0), "+v"(a1), "+v"(b1));
}
template <int CTL> __device__ __forceinline__ float fold_dpp(float lo, float hi, bool up) {
  return (up ? hi : lo) + dpp_mov<CTL>(up ? lo : hi);
}
// v[0..NV) (NV a power of two, 8..128) -> NV / 32 (at least 1) values per lane; lane_value gives their indexes.
template <int NV>
__device__ __forceinline__ void lane_sums(float (&v)[NV], int lane) {
#pragma unroll
  for (int i = 0; i < NV / 2; i += 2) {
    swap32(v[i], v[i + NV / 2], v[i + 1], v[i + 1 + NV / 2]);
    v[i] += v[i + NV / 2];
    v[i + 1] += v[i + 1 + NV / 2];
  }
#pragma unroll
  for (int i = 0; i < NV / 4; i += 2) {
    swap16(v[i], v[i + NV / 4], v[i + 1], v[i + 1 + NV / 4]);
    v[i] += v[i + NV / 4];
    v[i + 1] += v[i + 1 + NV / 4];
  }
  const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2;
#pragma unroll
  for (int i = 0; i < NV / 8; i++) v[i] = fold_dpp<0x128>(v[i], v[i + NV / 8], b3);  // lane ^ 8
  if constexpr (NV >= 16) {
#pragma unroll
    for (int i = 0; i < NV / 16; i++) v[i] = fold_dpp<0x141>(v[i], v[i + NV / 16], b2);  // lane ^ 7
  } else {
    v[0] += dpp_mov<0x141>(v[0]);
  }
  if constexpr (NV >= 32) {
#pragma unroll
    for (int i = 0; i < NV / 32; i++) v[i] = fold_dpp<0x4E>(v[i], v[i + NV / 32], b1);  // lane ^ 2
  } else {
    v[0] += dpp_mov<0x4E>(v[0]);
  }
#pragma unroll
  for (int i = 0; i < (NV >= 32 ? NV / 32 : 1); i++) v[i] += dpp_mov<0xB1>(v[i]);  // lane ^ 1
}
// Index of the value that register i of a lane holds after lane_sums, and whether the lane is the one to write it.
template <int NV>
__device__ __forceinline__ int lane_value(int i, int lane, bool& mine) {
  int k = i;
  k += ((lane >> 5) & 1) * (NV / 2) + ((lane >> 4) & 1) * (NV / 4) + ((lane >> 3) & 1) * (NV / 8);
  mine = (lane & 1) == 0;
  if (NV >= 16) k += ((lane >> 2) & 1) * (NV / 16);
  else mine = mine && !(lane & 4);
  if (NV >= 32) k += ((lane >> 1) & 1) * (NV / 32);
  else mine = mine && !(lane & 2);
  return k;
}

// d/dv of v sigma(v)
__device__ __forceinline__ float dsilu(float v, float s) { return s * fmaf(v, 1.f - s, 1.f); }

// The adjoint that a chunk alone sends back past its first step (its own outputs only).
template <typename T, int NS>
__global__ void __launch_bounds__(256) k_ssm_bwd_local(Args a, GradArgs ga) {
  __shared__ __attribute__((aligned(16))) float sbc[kSteps * 2 * NS];
  const Place pl = place(a, blockIdx.x);
  const long b = pl.b, c = pl.c;
  const long tbeg = pl.s * a.chunk, tend = min(a.T, tbeg + a.chunk);
  float A2[NS], g[NS];
#pragma unroll
  for (int n = 0; n < NS; n++) {
    A2[n] = n < a.N ? a.A[c * a.N + n] * kLog2e : 0.f;
    g[n] = 0.f;
  }
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.f;
  float dsum = 0.f;
  bool cleared = false;
  const T* dp = (const T*)a.delta + b * a.d_b + c;
  const T* zp = (const T*)a.z + (a.z ? b * a.z_b + c : 0);
  const T* gp = (const T*)ga.dy + b * ga.dy_b + c;
  for (long t0 = tbeg + (tend - tbeg - 1) / kSteps * kSteps; t0 >= tbeg; t0 -= kSteps) {
    float rd[kSteps], rz[kSteps], rg[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const long t = min(t0 + i, tend - 1);
      rd[i] = ldf(dp + t * a.d_t);
      rz[i] = a.z ? ldf(zp + t * a.z_t) : 0.f;
      rg[i] = ldf(gp + t * ga.dy_t);
    }
    __syncthreads();
    stage_bc<T, NS>(sbc, a, t0, tend, b, pl.g);
    __syncthreads();
#pragma unroll
    for (int i = kSteps - 1; i >= 0; i--) {
      const long t = t0 + i;
      if (t >= tend) continue;
      const float d = softplus(rd[i] + bias), dout = a.z ? rg[i] * silu(rz[i]) : rg[i];
      dsum += d;
      const bool st = starts(a, t, b);
      cleared |= st;
#pragma unroll
      for (int n = 0; n < NS; n++) {
        const float gn = fmaf(dout, sbc[(i * 2 + 1) * NS + n], g[n]);
        g[n] = st ? 0.f : ex2(d * A2[n]) * gn;
      }
    }
  }
  if (!pl.in) return;
  store_state<NS>(ga.carry + (pl.s * a.B * a.C + b * a.C + c) * a.N, g, a.N);
  a.dsum[(pl.s * a.B + b) * a.C + c] = cleared ? -1.f : dsum;
}

// Joins them from the end: carry[s] becomes the adjoint that comes in at chunk s's last step.
__global__ void __launch_bounds__(256) k_ssm_bwd_join(Args a, GradArgs ga) {
  const long BCN = a.B * a.C * a.N, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= BCN) return;
  const long bc = i / a.N, c = bc % a.C, n = i % a.N;
  const float A2 = a.A[c * a.N + n] * kLog2e;
  float run = 0.f;
  for (long s = a.chunks - 1; s >= 0; s--) {
    const float loc = ga.carry[s * BCN + i], d = a.dsum[s * a.B * a.C + bc];
    ga.carry[s * BCN + i] = run;
    run = d < 0.f ? loc : fmaf(ex2(A2 * d), run, loc);
  }
}

// The gradient of one chunk after another. Batches of kS = keep_steps(NS) steps run backwards in time; each restores the
// kept state before it, runs its steps forward again keeping a_t h_{t-1} of every step in registers, then runs them
// backwards: g_t = C_t dout_t + a_{t+1} g_{t+1}. The sums over channels (dB, dC) are folded over the wavefront's lanes
// and added over the block's wavefronts in LDS; the parameters' gradients stay in registers over all chunks of
// the block. A block takes the items row, row + rows, ... of its channel block, an item being a chunk of a sequence.
template <typename T, int NS>
__global__ void __launch_bounds__(64 * bwd_waves(NS)) k_ssm_bwd(Args a, GradArgs ga) {
  constexpr int kS = keep_steps(NS), NV = 2 * NS;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  float* sbc = lds;                  // [kS][2][NS]
  float* red = lds + kS * NV;        // [waves][kS][2][NS]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const long G = a.C / a.per;
  const int cb = (int)(blockIdx.x % a.blocks_c);
  const int grp = (int)((blockIdx.x / a.blocks_c) % G);
  const long row = blockIdx.x / (a.blocks_c * G);
  const long lc = (long)cb * blockDim.x + threadIdx.x;
  const bool in = lc < a.per;
  const long c = grp * a.per + (in ? lc : a.per - 1);
  Conv cv;
  cv.init(a, c);
  float A2[NS], dA[NS], g[NS];
#pragma unroll
  for (int n = 0; n < NS; n++) {
    A2[n] = n < a.N ? a.A[c * a.N + n] * kLog2e : 0.f;
    dA[n] = 0.f;
  }
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
  float dD = 0.f, dbias = 0.f, dcb = 0.f, dw[kTaps] = {};
  const int K = cv.K;
  for (long item = row; item < a.B * a.chunks; item += ga.rows) {
    const long b = item % a.B, s = item / a.B;
    const long tbeg = s * a.chunk, tend = min(a.T, tbeg + a.chunk);
    const long hoff = (b * a.C + c) * a.N;
    if (a.chunks > 1) load_state<NS>(g, ga.carry + s * a.B * a.C * a.N + hoff, a.N);
    else {
#pragma unroll
      for (int n = 0; n < NS; n++) g[n] = 0.f;
    }
    // ds of the three steps after the current one, of the same episode (zero past the chunk: its successor's
    // share of this chunk's last steps comes through the halo)
    float q1 = 0.f, q2 = 0.f, q3 = 0.f;
    const T* xp = (const T*)a.x + b * a.x_b + c;
    const T* dp = (const T*)a.delta + b * a.d_b + c;
    const T* zp = (const T*)a.z + (a.z ? b * a.z_b + c : 0);
    const T* gp = (const T*)ga.dy + b * ga.dy_b + c;
    for (long t0 = tbeg + (tend - tbeg - 1) / kS * kS; t0 >= tbeg; t0 -= kS) {
      float rx[kS], rd[kS], rz[kS], rg[kS];
#pragma unroll
      for (int i = 0; i < kS; i++) {
        const long t = min(t0 + i, tend - 1);
        rx[i] = ldf(xp + t * a.x_t);
        rd[i] = ldf(dp + t * a.d_t) + bias;
        rz[i] = a.z ? ldf(zp + t * a.z_t) : 0.f;
        rg[i] = ldf(gp + t * ga.dy_t);
      }
      float h[NS], ah[kS][NS];
      load_state<NS>(h, ga.keep + (t0 / kS) * a.B * a.C * a.N + hoff, a.N);
      cv.clear();
      conv_seek<T>(cv, a, t0, b, c);
      __syncthreads();  // the last batch's sums have been read
      for (int e = threadIdx.x; e < kS * NV; e += blockDim.x) {
        const int n = e % NS, which = (e / NS) & 1;
        const long t = t0 + e / NV;
        float v = 0.f;
        if (n < a.N && t < tend) {
          const long col = grp * a.N + n;
          v = which ? ldf((const T*)a.Cm + t * a.cm_t + b * a.cm_b + col)
                    : ldf((const T*)a.Bm + t * a.bm_t + b * a.bm_b + col);
        }
        sbc[e] = v;
      }
      __syncthreads();
      // forward again
      float pre[kS], u[kS], d[kS], p1[kS], p2[kS], p3[kS];
      bool st[kS];
#pragma unroll
      for (int i = 0; i < kS; i++) {
        const long t = t0 + i;
        st[i] = t < tend && starts(a, t, b);
        if (st[i]) cv.clear();
        pre[i] = K ? cv.pre(rx[i]) : rx[i];
        u[i] = K ? silu(pre[i]) : rx[i];
        p1[i] = cv.p[2];
        p2[i] = cv.p[1];
        p3[i] = cv.p[0];
        cv.push(rx[i]);
        d[i] = softplus(rd[i]);
        const float du = d[i] * u[i];
#pragma unroll
        for (int n = 0; n < NS; n++) {
          ah[i][n] = st[i] ? 0.f : ex2(d[i] * A2[n]) * h[n];
          h[n] = fmaf(du, sbc[i * NV + n], ah[i][n]);
        }
      }
      // and back
#pragma unroll
      for (int i = kS - 1; i >= 0; i--) {
        const long t = t0 + i;
        if (t >= tend) {
          if (lane < NV) red[(wave * kS + i) * NV + lane] = 0.f;
          continue;
        }
        const float sz = a.z ? sigm(rz[i]) : 0.f;
        const float dout = a.z ? rg[i] * (rz[i] * sz) : rg[i];
        const float du = d[i] * u[i];
        float o = Dc * u[i], gB = 0.f, Aq = 0.f;
        float v[NV];
#pragma unroll
        for (int n = 0; n < NS; n++) {
          const float Bn = sbc[i * NV + n], Cn = sbc[i * NV + NS + n];
          const float hn = fmaf(du, Bn, ah[i][n]);
          const float gn = fmaf(dout, Cn, g[n]);
          o = fmaf(hn, Cn, o);
          gB = fmaf(gn, Bn, gB);
          const float q = gn * ah[i][n];
          Aq = fmaf(A2[n], q, Aq);
          dA[n] = fmaf(d[i], q, dA[n]);
          v[n] = in ? gn * du : 0.f;
          v[NS + n] = in ? hn * dout : 0.f;
          g[n] = st[i] ? 0.f : ex2(d[i] * A2[n]) * gn;
        }
        lane_sums<NV>(v, lane);
#pragma unroll
        for (int k = 0; k < (NV >= 32 ? NV / 32 : 1); k++) {
          bool mine;
          const int idx = lane_value<NV>(k, lane, mine);
          if (mine) red[(wave * kS + i) * NV + idx] = v[k];
        }
        const float ddt = fmaf(u[i], gB, Aq * (1.f / kLog2e)) * sigm(rd[i]);
        float ds = fmaf(d[i], gB, Dc * dout);
        dD = fmaf(dout, u[i], dD);
        dbias += ddt;
        float dxv = ds;
        if (K) {
          const float sg = sigm(pre[i]);
          ds *= dsilu(pre[i], sg);
          dcb += ds;
          dw[3] = fmaf(ds, rx[i], dw[3]);
          dw[2] = fmaf(ds, p1[i], dw[2]);
          dw[1] = fmaf(ds, p2[i], dw[1]);
          dw[0] = fmaf(ds, p3[i], dw[0]);
          dxv = fmaf(cv.w[3], ds, fmaf(cv.w[2], q1, fmaf(cv.w[1], q2, cv.w[0] * q3)));
          q3 = st[i] || K < 4 ? 0.f : q2;
          q2 = st[i] || K < 3 ? 0.f : q1;
          q1 = st[i] || K < 2 ? 0.f : ds;
        }
        if (in) {
          if (ga.ddelta) stf((T*)ga.ddelta + t * ga.dd_t + b * ga.dd_b + c, ddt);
          if (a.z && ga.dz) stf((T*)ga.dz + t * ga.dz_t + b * ga.dz_b + c, rg[i] * o * dsilu(rz[i], sz));
          // the last K - 1 steps of a chunk that has a successor are finished by the halo's launch
          if (ga.dx) {
            if (t >= tend - (K - 1) && tend < a.T) ga.halo[(((s * 2) * a.B + b) * (kTaps - 1) + (tend - 1 - t)) * a.C + c] = dxv;
            else stf((T*)ga.dx + t * ga.dx_t + b * ga.dx_b + c, dxv);
          }
        }
      }
      __syncthreads();
      // the block's sums over its wavefronts, in order
      for (int e = threadIdx.x; e < kS * NV; e += blockDim.x) {
        const int n = e % NS, which = (e / NS) & 1;
        const long t = t0 + e / NV;
        if (n >= a.N || t >= tend) continue;
        float sum = 0.f;
        for (int w = 0; w < waves; w++) sum += red[w * kS * NV + e];
        if (ga.bc) ga.bc[((((long)cb * a.T + t) * a.B + b) * G + grp) * 2 * a.N + which * a.N + n] = sum;
        else if (which && ga.dC) stf((T*)ga.dC + t * ga.dc_t + b * ga.dc_b + grp * a.N + n, sum);
        else if (!which && ga.dB) stf((T*)ga.dB + t * ga.db_t + b * ga.db_b + grp * a.N + n, sum);
      }
    }
    // what this chunk adds to dx of the K - 1 steps before it: step tbeg - 1 - j takes ds of up to K - 1 - j steps on
    if (in && K > 1 && s > 0 && ga.dx) {
      const float hq[kTaps - 1] = {fmaf(cv.w[2], q1, fmaf(cv.w[1], q2, cv.w[0] * q3)), fmaf(cv.w[1], q1, cv.w[0] * q2),
                                   cv.w[0] * q1};
#pragma unroll
      for (int j = 0; j < kTaps - 1; j++)
        if (j < K - 1) ga.halo[(((s * 2 - 1) * a.B + b) * (kTaps - 1) + j) * a.C + c] = hq[j];
    }
  }
  if (in && ga.par) {
    float* p = ga.par + (row * a.C + c) * ga.P;
#pragma unroll
    for (int n = 0; n < NS; n++)
      if (n < a.N) p[n] = dA[n];
    p += a.N;
    p[0] = dD;
    p[1] = dbias;
    p[2] = dcb;
#pragma unroll
    for (int k = 0; k < kTaps; k++)
      if (k >= kTaps - K) p[3 + k - (kTaps - K)] = dw[k];
  }
}

// dx of the last K - 1 steps of every chunk but the last: the chunk's own part plus its successor's, unless an
// episode starts in between (the successor's part then is zero already, and the own part stopped at the start).
template <typename T>
__global__ void __launch_bounds__(256) k_ssm_halo(Args a, GradArgs ga) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, K1 = a.K - 1;
  if (i >= (a.chunks - 1) * a.B * K1 * a.C) return;
  const long c = i % a.C, j = i / a.C % K1, b = i / (a.C * K1) % a.B, s = i / (a.C * K1 * a.B);
  const long tend = (s + 1) * a.chunk, t = tend - 1 - j;
  float v = ga.halo[(((s * 2) * a.B + b) * (kTaps - 1) + j) * a.C + c];
  // an episode that starts at a step after t and before tend cuts this step off from the successor
  bool cut = false;
  for (long q = t + 1; q < tend; q++) cut |= starts(a, q, b);
  if (!cut) v += ga.halo[(((s * 2 + 1) * a.B + b) * (kTaps - 1) + j) * a.C + c];
  stf((T*)ga.dx + t * ga.dx_t + b * ga.dx_b + c, v);
}

// dB, dC = the channel blocks' sums in order.
template <typename T>
__global__ void __launch_bounds__(256) k_ssm_fold_bc(Args a, GradArgs ga) {
  const long G = a.C / a.per, W = G * 2 * a.N, tot = a.T * a.B * W;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < tot; i += (long)gridDim.x * 256) {
    const long tb = i / W, b = tb % a.B, t = tb / a.B;
    const long e = i % W, g = e / (2 * a.N), r = e % (2 * a.N), which = r / a.N, n = r % a.N;
    float s = 0.f;
    for (int cb = 0; cb < a.blocks_c; cb++) s += ga.bc[cb * tot + i];
    if (which) {
      if (ga.dC) stf((T*)ga.dC + t * ga.dc_t + b * ga.dc_b + g * a.N + n, s);
    } else if (ga.dB) {
      stf((T*)ga.dB + t * ga.db_t + b * ga.db_b + g * a.N + n, s);
    }
  }
}

struct ParOut {
  float *dA, *dD, *dbias, *dcw, *dcb;
};
// The parameters' gradients: the rows' sums in a fixed order, four ranges of rows per value.
__global__ void __launch_bounds__(256) k_ssm_fold_par(const float* __restrict__ par, long rows, long CP, int N, int K, int P,
                                                      ParOut o) {
  __shared__ float sh[4][64];
  const int e = threadIdx.x & 63, z = threadIdx.x >> 6;
  const long i = (long)blockIdx.x * 64 + e;
  const long per = (rows + 3) / 4, end = min(rows, (z + 1) * per);
  float s = 0.f;
  if (i < CP) {
    long r = z * per;
    for (; r + 8 <= end; r += 8) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; q++) v[q] = par[(r + q) * CP + i];
#pragma unroll
      for (int q = 0; q < 8; q++) s += v[q];
    }
    for (; r < end; r++) s += par[r * CP + i];
  }
  sh[z][e] = s;
  __syncthreads();
  if (z || i >= CP) return;
  s = (sh[0][e] + sh[1][e]) + (sh[2][e] + sh[3][e]);
  const long c = i / P;
  const int k = (int)(i % P);
  if (k < N) {
    if (o.dA) o.dA[c * N + k] = s;
  } else if (k == N) {
    if (o.dD) o.dD[c] = s;
  } else if (k == N + 1) {
    if (o.dbias) o.dbias[c] = s;
  } else if (k == N + 2) {
    if (o.dcb) o.dcb[c] = s;
  } else if (o.dcw) {
    o.dcw[c * K + k - N - 3] = s;
  }
}

// ---- host ----------------------------------------------------------------------------------------------
int check(const ph_ssm_args& p, const char* who) {
  PH_REQUIRE(p.dtype == PH_F32 || p.dtype == PH_BF16, "%s: dtype must be F32 or BF16", who);
  PH_REQUIRE(p.C >= 1 && p.C <= (1u << 24) && p.N >= 1 && p.N <= (size_t)kMaxStates, "%s: C = %zu channels of N = %zu states (N <= 64)",
             who, p.C, p.N);
  PH_REQUIRE(p.T <= (1u << 30) && p.B <= (1u << 24) && p.B * p.C <= (1ull << 32), "%s: T = %zu, B = %zu, C = %zu out of range",
             who, p.T, p.B, p.C);
  PH_REQUIRE(p.G >= 1 && p.C % p.G == 0, "%s: %zu groups do not divide %zu channels", who, p.G, p.C);
  PH_REQUIRE(p.K <= (size_t)kTaps, "%s: K = %zu taps (at most 4)", who, p.K);
  PH_REQUIRE(!p.K || p.conv_w, "%s: conv_w missing", who);
  if (p.T == 0 || p.B == 0) return PH_OK;
  PH_REQUIRE(p.x && p.delta && p.Bm && p.Cm && p.A, "%s: x, delta, B, C or A missing", who);
  return PH_OK;
}

Args args_of(const ph_ssm_args& p) {
  Args a{};
  a.T = (long)p.T; a.B = (long)p.B; a.C = (long)p.C; a.N = (long)p.N; a.per = (long)(p.C / p.G); a.K = (long)p.K;
  a.x = p.x; a.z = p.z; a.delta = p.delta; a.Bm = p.Bm; a.Cm = p.Cm;
  a.x_t = p.x_t; a.x_b = p.x_b; a.z_t = p.z_t; a.z_b = p.z_b; a.d_t = p.delta_t; a.d_b = p.delta_b;
  a.bm_t = p.Bm_t; a.bm_b = p.Bm_b; a.cm_t = p.Cm_t; a.cm_b = p.Cm_b;
  a.A = p.A; a.D = p.D; a.dt_bias = p.dt_bias; a.conv_w = p.conv_w; a.conv_b = p.conv_b;
  a.done = p.done; a.first = p.first; a.h0 = p.h0; a.win0 = p.win0;
  return a;
}

// Threads of a block: whole wavefronts over a group's channels, `most` at most.
int block_threads(const Args& a, int most) {
  const long w = (a.per + 63) / 64;
  return 64 * (int)(w < most ? w : most);
}

// Chunks of time: enough wavefronts for every SIMD to hold two, in chunks of at least 32 steps.
void set_chunks(Args& a) {
  const long waves = a.B * (a.C / a.per) * ((a.per + 63) / 64);
  long want = (2048 + waves - 1) / waves;
  const long most = (a.T + 31) / 32;
  if (want > most) want = most;
  if (want < 1) want = 1;
  a.chunk = (a.T + want - 1) / want;
  a.chunk = (a.chunk + kSteps - 1) / kSteps * kSteps;
  a.chunks = (a.T + a.chunk - 1) / a.chunk;
}

template <typename T, int NS>
int fwd_n(Args& a, float* win_out, hipStream_t st) {
  const int nt = block_threads(a, 4);
  a.blocks_c = (int)((a.per + nt - 1) / nt);
  const long blocks = a.chunks * a.B * (a.C / a.per) * a.blocks_c;
  if (a.chunks > 1) {
    k_ssm_fwd<T, NS, true><<<(unsigned)blocks, nt, 0, st>>>(a);
    PH_LAUNCH_CHECK();
    k_ssm_join<<<ceil_div((size_t)(a.B * a.C * a.N), 256), 256, 0, st>>>(a);
    PH_LAUNCH_CHECK();
  }
  k_ssm_fwd<T, NS, false><<<(unsigned)blocks, nt, 0, st>>>(a);
  PH_LAUNCH_CHECK();
  if (win_out && a.K > 1) {
    k_ssm_window<T><<<ceil_div((size_t)(a.B * a.C), 256), 256, 0, st>>>(a, win_out);
    PH_LAUNCH_CHECK();
  }
  return PH_OK;
}

template <typename T>
int fwd_t(Args& a, float* win_out, hipStream_t st) {
  switch (states_of(a.N)) {
    case 4: return fwd_n<T, 4>(a, win_out, st);
    case 8: return fwd_n<T, 8>(a, win_out, st);
    case 16: return fwd_n<T, 16>(a, win_out, st);
    case 32: return fwd_n<T, 32>(a, win_out, st);
    default: return fwd_n<T, 64>(a, win_out, st);
  }
}

template <typename T, int NS>
int bwd_n(Args& a, GradArgs& ga, const ParOut& po, hipStream_t st) {
  constexpr int kS = keep_steps(NS);
  const int nl = block_threads(a, 4), nt = block_threads(a, bwd_waves(NS));
  const long G = a.C / a.per;
  if (a.chunks > 1) {
    a.blocks_c = (int)((a.per + nl - 1) / nl);
    k_ssm_bwd_local<T, NS><<<(unsigned)(a.chunks * a.B * G * a.blocks_c), nl, 0, st>>>(a, ga);
    PH_LAUNCH_CHECK();
    k_ssm_bwd_join<<<ceil_div((size_t)(a.B * a.C * a.N), 256), 256, 0, st>>>(a, ga);
    PH_LAUNCH_CHECK();
  }
  a.blocks_c = (int)((a.per + nt - 1) / nt);
  const size_t lds = (size_t)(1 + nt / 64) * kS * 2 * NS * 4;
  static_assert((1 + bwd_waves(NS)) * kS * 2 * NS * 4 <= kMaxLdsBytes, "LDS budget");
  k_ssm_bwd<T, NS><<<(unsigned)(ga.rows * G * a.blocks_c), nt, lds, st>>>(a, ga);
  PH_LAUNCH_CHECK();
  if (a.chunks > 1 && a.K > 1 && ga.dx) {
    k_ssm_halo<T><<<ceil_div((size_t)((a.chunks - 1) * a.B * (a.K - 1) * a.C), 256), 256, 0, st>>>(a, ga);
    PH_LAUNCH_CHECK();
  }
  if (ga.bc) {
    const size_t n = (size_t)a.T * a.B * G * 2 * a.N;
    const unsigned blocks = ceil_div(n, 256);
    k_ssm_fold_bc<T><<<blocks < 8192 ? blocks : 8192, 256, 0, st>>>(a, ga);
    PH_LAUNCH_CHECK();
  }
  const long CP = a.C * ga.P;
  k_ssm_fold_par<<<ceil_div((size_t)CP, 64), 256, 0, st>>>(ga.par, ga.rows, CP, (int)a.N, (int)a.K, ga.P, po);
  PH_LAUNCH_CHECK();
  return PH_OK;
}

template <typename T>
int bwd_t(Args& a, GradArgs& ga, const ParOut& po, hipStream_t st) {
  switch (states_of(a.N)) {
    case 4: return bwd_n<T, 4>(a, ga, po, st);
    case 8: return bwd_n<T, 8>(a, ga, po, st);
    case 16: return bwd_n<T, 16>(a, ga, po, st);
    case 32: return bwd_n<T, 32>(a, ga, po, st);
    default: return bwd_n<T, 64>(a, ga, po, st);
  }
}

template <typename T, bool VEC>
int step_t(const Args& a, float* h, float* win, hipStream_t st) {
  const int lpc = states_of(a.N) / 4;
  const unsigned grid = (unsigned)((a.C + 256 / lpc - 1) / (256 / lpc) * a.B);
  switch (lpc) {
    case 1: k_ssm_step<T, 1, VEC><<<grid, 256, 0, st>>>(a, h, win); break;
    case 2: k_ssm_step<T, 2, VEC><<<grid, 256, 0, st>>>(a, h, win); break;
    case 4: k_ssm_step<T, 4, VEC><<<grid, 256, 0, st>>>(a, h, win); break;
    case 8: k_ssm_step<T, 8, VEC><<<grid, 256, 0, st>>>(a, h, win); break;
    default: k_ssm_step<T, 16, VEC><<<grid, 256, 0, st>>>(a, h, win); break;
  }
  PH_LAUNCH_CHECK();
  return PH_OK;
}

__global__ void __launch_bounds__(256) k_ssm_zero(ParOut o, int C, int N, int K) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < C * N; i += gridDim.x * 256) {
    if (o.dA) o.dA[i] = 0.f;
    if (i < C) {
      if (o.dD) o.dD[i] = 0.f;
      if (o.dbias) o.dbias[i] = 0.f;
      if (o.dcb) o.dcb[i] = 0.f;
      for (int k = 0; k < K; k++)
        if (o.dcw) o.dcw[i * K + k] = 0.f;
    }
  }
}

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" size_t ph_ssm_keep_floats(const ph_ssm_args* p) {
  if (!p || p->N < 1 || p->N > (size_t)kMaxStates) return 0;
  const size_t ks = (size_t)keep_steps(states_of((long)p->N));
  return (p->T + ks - 1) / ks * p->B * p->C * p->N;
}

extern "C" int ph_ssm_scan(const ph_ssm_args* p, void* y, long y_t, long y_b, float* h_out, float* win_out, float* keep,
                           void* stream) {
  PH_REQUIRE(p, "ssm_scan: arguments missing");
  PH_TRY(check(*p, "ssm_scan"));
  if (p->B == 0) return PH_OK;
  PH_REQUIRE(p->T >= 1, "ssm_scan: no steps");
  PH_REQUIRE(y, "ssm_scan: y missing");
  hipStream_t st = as_stream(stream);
  Args a = args_of(*p);
  a.y = y; a.y_t = y_t; a.y_b = y_b; a.h_out = h_out; a.keep = keep;
  set_chunks(a);
  if (a.chunks > 1) {
    const size_t nh = (size_t)a.chunks * a.B * a.C * a.N, nd = (size_t)a.chunks * a.B * a.C;
    float* ws = (float*)scratch(kSlotSsm, (nh + nd) * 4);
    if (!ws) return PH_ERR_NOMEM;
    a.hloc = ws;
    a.dsum = ws + nh;
  }
  return p->dtype == PH_BF16 ? fwd_t<uint16_t>(a, win_out, st) : fwd_t<float>(a, win_out, st);
}

extern "C" int ph_ssm_scan_grad(const ph_ssm_args* p, const float* keep, const void* dy, long dy_t, long dy_b,
                                const ph_ssm_grads* g, void* stream) {
  PH_REQUIRE(p && g, "ssm_scan_grad: arguments missing");
  PH_TRY(check(*p, "ssm_scan_grad"));
  hipStream_t st = as_stream(stream);
  const ParOut po{g->dA, g->dD, g->ddt_bias, g->dconv_w, g->dconv_b};
  if (p->B == 0) {  // no sequences: the parameters' sums are zero
    k_ssm_zero<<<256, 256, 0, st>>>(po, (int)p->C, (int)p->N, (int)p->K);
    PH_LAUNCH_CHECK();
    return PH_OK;
  }
  PH_REQUIRE(p->T >= 1, "ssm_scan_grad: no steps");
  PH_REQUIRE(dy && keep, "ssm_scan_grad: dy or the kept states missing");
  Args a = args_of(*p);
  set_chunks(a);
  GradArgs ga{};
  ga.dy = dy; ga.dy_t = dy_t; ga.dy_b = dy_b; ga.keep = keep;
  ga.dx = g->dx; ga.dx_t = g->dx_t; ga.dx_b = g->dx_b;
  ga.dz = g->dz; ga.dz_t = g->dz_t; ga.dz_b = g->dz_b;
  ga.ddelta = g->ddelta; ga.dd_t = g->ddelta_t; ga.dd_b = g->ddelta_b;
  ga.dB = g->dBm; ga.db_t = g->dBm_t; ga.db_b = g->dBm_b;
  ga.dC = g->dCm; ga.dc_t = g->dCm_t; ga.dc_b = g->dCm_b;
  ga.P = (int)(a.N + a.K + 3);
  const long G = a.C / a.per, nt = block_threads(a, bwd_waves(states_of(a.N))), bc = (a.per + nt - 1) / nt;
  // blocks of a channel block: a few for every CU, each with many items of its own
  const long items = a.B * a.chunks;
  ga.rows = 1024 / (G * bc);
  if (ga.rows > items) ga.rows = items;
  if (ga.rows < 1) ga.rows = 1;
  const size_t nh = a.chunks > 1 ? (size_t)a.chunks * a.B * a.C * a.N : 0, nd = a.chunks > 1 ? (size_t)a.chunks * a.B * a.C : 0;
  const size_t nhalo = a.chunks > 1 ? (size_t)(2 * a.chunks) * a.B * (kTaps - 1) * a.C : 0;
  const size_t nbc = bc > 1 && (ga.dB || ga.dC) ? (size_t)bc * a.T * a.B * G * 2 * a.N : 0;
  const size_t npar = (size_t)ga.rows * a.C * ga.P;
  float* ws = (float*)scratch(kSlotSsm, (nh + nd + nhalo + nbc + npar) * 4);
  if (!ws) return PH_ERR_NOMEM;
  ga.carry = ws;
  a.dsum = ws + nh;
  ga.halo = ws + nh + nd;
  ga.bc = nbc ? ws + nh + nd + nhalo : nullptr;
  ga.par = ws + nh + nd + nhalo + nbc;
  return p->dtype == PH_BF16 ? bwd_t<uint16_t>(a, ga, po, st) : bwd_t<float>(a, ga, po, st);
}

extern "C" int ph_ssm_step(const ph_ssm_args* p, void* y, long y_b, float* h, float* win, void* stream) {
  PH_REQUIRE(p, "ssm_step: arguments missing");
  PH_REQUIRE(p->T <= 1, "ssm_step: T = %zu (a single step)", p->T);
  PH_TRY(check(*p, "ssm_step"));
  if (p->T == 0 || p->B == 0) return PH_OK;
  PH_REQUIRE(y && h, "ssm_step: y or the state missing");
  PH_REQUIRE(p->K < 2 || win, "ssm_step: the convolution's window missing");
  Args a = args_of(*p);
  a.y = y; a.y_b = y_b;
  const bool vec = p->N % 4 == 0 && ((uintptr_t)h % 16) == 0 && ((uintptr_t)p->A % 16) == 0 &&
                   (states_of((long)p->N) == (long)p->N);
  hipStream_t st = as_stream(stream);
  if (p->dtype == PH_BF16) return vec ? step_t<uint16_t, true>(a, h, win, st) : step_t<uint16_t, false>(a, h, win, st);
  return vec ? step_t<float, true>(a, h, win, st) : step_t<float, false>(a, h, win, st);
}
