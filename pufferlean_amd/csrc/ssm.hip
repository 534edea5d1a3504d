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
// Layout. A lane owns one channel, a wavefront 64 channels of one sequence, so the only values that cross lanes are
// B_t and C_t, which every lane of the block reads from LDS as broadcasts (staged there kSteps steps at a time,
// converted once). Within those steps the states are taken four at a time: a lane's four states and decays rest in
// LDS slots of its own and are in registers for the kSteps steps. So any N runs in the same few registers and short
// code, and the state is fp32 throughout and never written per step. What a step costs is vector arithmetic: per state
// one exponential (8 cycles of a wavefront), the decay's argument, the input, the update and the output (4 cycles each),
// 24 cycles in all against 8 bytes of memory per channel and step; the gradient takes about three times as many.
//
// Measured, bf16, 16 states, four taps, gated: 64 steps of 2048 sequences x 512 channels forward 373 us, of which vector
// instructions issue 70 % (the states' own 24 cycles would be 164 us), gradient 1139 us, 73 %; 8192 steps of 2 sequences
// x 512 channels 102 us; 2048 steps of 8 x 384, two groups, both directions 313 us. What is left of the time is
// wavefronts that wait: two on a SIMD in the gradient (its registers), four forward (its LDS slots).
//
// Long sequences of few channels do not fill the chip with one wavefront per 64 channels, so time is cut into
// chunks: a first launch runs every chunk from a zero state and keeps its end state and the sum of d_t (the
// chunk's decay is exp(A sum d)), a second joins the chunks' start states in order, and the third runs the
// chunks again from those.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "routes.hpp"

#include <type_traits>

namespace ph {
namespace {

constexpr int kSteps = kSsmSteps;  // steps of a batch: staged and loaded together, and between two kept states of the training forward
constexpr int kTaps = 4;   // most taps of the convolution; fewer are padded with zero taps in front
constexpr int kMaxStates = 64;
constexpr float kLog2e = 1.4426950408889634f;

// Global pointers as such: the compiler loses track of a pointer that an asm has touched (walk, below) and would access it
// as one that may also point to LDS.
#define PH_GLOBAL __attribute__((address_space(1)))
template <typename T> using gin = const PH_GLOBAL T*;
template <typename T> using gout = PH_GLOBAL T*;
typedef float f4t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f4t f4(float x, float y, float z, float w) { return f4t{x, y, z, w}; }

struct Args {
  int T, C, N, per, K;  // per: channels of a group
  int Q;                // states in fours, N rounded up
  long B;
  const void *x, *z, *delta, *Bm, *Cm;
  long x_t, x_b, z_t, z_b, d_t, d_b, bm_t, bm_b, cm_t, cm_b;
  const float *A, *D, *dt_bias, *conv_w, *conv_b;
  const float *done, *first, *h0, *win0;
  void* y;
  long y_t, y_b;
  float *h_out, *keep, *win_out;
  int win_here;         // the scan's last chunk writes win_out
  int chunk, chunks;    // steps of a chunk (a multiple of kSteps), their number
  float *hloc, *dsum;   // [chunks] end (then start) states, [chunks][B][C] sums of d (-1: cleared inside)
  unsigned blocks_c, G; // channel blocks of a group, groups
};
// The library's own states are [..][B][Q][C][4]: a wavefront moves four states of 64 channels as 1 KB. The caller's are
// [B][C][N].

__device__ __forceinline__ float ldf(gin<uint16_t> p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float ldf(gin<float> p) { return *p; }
__device__ __forceinline__ float ldf(const uint16_t* p) { return ldf((gin<uint16_t>)p); }
__device__ __forceinline__ float ldf(const float* p) { return ldf((gin<float>)p); }
__device__ __forceinline__ float raw_f32(float v) { return v; }
__device__ __forceinline__ float raw_f32(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ void stf(gout<uint16_t> p, float v) { *p = bf16_rne(v); }
__device__ __forceinline__ void stf(gout<float> p, float v) { *p = v; }

__device__ __forceinline__ float ex2(float v) { return __builtin_amdgcn_exp2f(v); }
// softplus, max(v, 0) + log(1 + e) with e = exp(-|v|). What rounding 1 + e to w dropped, e - (w - 1), is added back as it is
// (its share of the logarithm is that over w, and it is nothing but where w is near 1), so small e keep their digits.
__device__ __forceinline__ float softplus(float v) {
  const float e = ex2(-fabsf(v) * kLog2e), w = 1.f + e;
  return fmaxf(v, 0.f) + fmaf(__builtin_amdgcn_logf(w), 1.f / kLog2e, e - (w - 1.f));
}
__device__ __forceinline__ float sigma(float v) { return __builtin_amdgcn_rcpf(1.f + ex2(v * -kLog2e)); }
__device__ __forceinline__ float silu(float v) { return v * sigma(v); }
// d/dv of v sigma(v), s = sigma(v)
__device__ __forceinline__ float dsilu(float v, float s) { return s * fmaf(v, 1.f - s, 1.f); }

// Whether step t of sequence b starts an episode.
__device__ __forceinline__ bool starts(const Args& a, int t, long b) {
  if (t > 0) return a.done && a.done[(long)(t - 1) * a.B + b] != 0.f;
  return t == 0 && a.first && a.first[b] != 0.f;
}
// Bit j of flag_bits(flag_load(..)): step t0 - 3 + j starts an episode (j < 11: a batch and the three steps that its
// convolutions look back to). One load per lane, one ballot, apart so that the load can be issued a batch ahead.
__device__ __forceinline__ float flag_load(const Args& a, int t0, int tend, long b) {
  int me = threadIdx.x;
  asm("" : "+v"(me));  // computed here, not once for all batches
  const int j = me & 63, t = t0 - (kTaps - 1) + j;
  float f = 0.f;
  if (j < kSteps + kTaps - 1 && t < tend && t >= 0) {
    if (t > 0) f = a.done ? a.done[(long)(t - 1) * a.B + b] : 0.f;
    else f = a.first ? a.first[b] : 0.f;
  }
  return f;
}
__device__ __forceinline__ unsigned flag_bits(float f) { return (unsigned)__ballot(f != 0.f); }

// The convolution of one channel, padded to four taps. Inputs that a step does not see (past its taps, or of the
// episode before) are selected away and not multiplied by zero: they may be infinite.
struct Conv {
  float w[kTaps], bias;
  int K;
  __device__ __forceinline__ void init(const Args& a, unsigned c) {
    K = a.K;
#pragma unroll
    for (int i = 0; i < kTaps; i++) {
      const int k = i - (kTaps - K);
      w[i] = K > 0 && k >= 0 ? a.conv_w[(long)c * K + k] : 0.f;
    }
    bias = K > 0 && a.conv_b ? a.conv_b[c] : 0.f;
  }
  // How many steps back step i of a batch sees (0..3), uniform.
  __device__ __forceinline__ int reach(unsigned bits, int i) const {
    const int n = K < 1 ? 0 : K - 1;
    if (bits >> i & 8u) return 0;
    if (bits >> i & 4u) return min(n, 1);
    if (bits >> i & 2u) return min(n, 2);
    return n;
  }
  __device__ __forceinline__ float pre(float x, float x1, float x2, float x3) const {
    return fmaf(w[3], x, fmaf(w[2], x1, fmaf(w[1], x2, fmaf(w[0], x3, bias))));
  }
};

// The three inputs before step t0 as bits of T (of the sequence, or as fp32 values of the carried window).
template <typename T>
__device__ __forceinline__ void look_back(float (&x)[kTaps - 1], const Args& a, int t0, long b, unsigned c) {
  const gin<T> p = (gin<T>)a.x + b * a.x_b;
  const int K1 = a.K - 1;
#pragma unroll
  for (int j = 0; j < kTaps - 1; j++) {
    const int t = t0 - (kTaps - 1) + j;
    x[j] = 0.f;
    if (t >= 0) x[j] = ldf(p + t * a.x_t + c);
    else if (K1 + t >= 0 && a.win0) x[j] = a.win0[(b * K1 + K1 + t) * a.C + c];
  }
}

// A lane's place in uniform rows of T. A 32-bit byte offset beside a scalar base is an address that loads and stores take as
// it is; but the compiler widens the offset once, outside the loops, and then adds in 64 bits for every row. What comes out of
// the empty asm it has to widen where it is used.
template <typename T>
struct Lane {
  unsigned o;
  __device__ __forceinline__ explicit Lane(unsigned c) : o(c * (unsigned)sizeof(T)) { asm("" : "+v"(o)); }
  __device__ __forceinline__ gin<T> operator()(gin<T> row) const { return (gin<T>)((gin<char>)row + o); }
  __device__ __forceinline__ gout<T> operator()(gout<T> row) const { return (gout<T>)((gout<char>)row + o); }
};

// A uniform row pointer that walks over steps. The empty asm keeps the walk a chain of scalar additions: without it the
// compiler forms the addresses of all of a batch's rows at once, hundreds of scalar registers that it then spills.
template <typename P>
__device__ __forceinline__ void walk(P& p, long d) {
  p += d;
  asm("" : "+s"(p));
}

// The kernel's own arguments, read again from where the launch put them: Args first, GradArgs behind. The compiler reads
// arguments once, at the kernel's start, and what the scalar registers cannot hold over the loops it keeps in lanes of
// vector registers, an instruction of each wavefront for every word it takes back.
template <typename A>
__device__ __forceinline__ A again(unsigned at) {
  static_assert(sizeof(A) % 8 == 0 && alignof(A) == 8, "read in words of eight bytes");
  auto p = (const __attribute__((address_space(4))) uint64_t*)__builtin_amdgcn_kernarg_segment_ptr();
  asm("" : "+s"(p));
  uint64_t w[sizeof(A) / 8];
#pragma unroll
  for (unsigned i = 0; i < sizeof(A) / 8; i++) w[i] = p[at / 8 + i];
  return __builtin_bit_cast(A, w);
}

// A value that every lane holds, in a scalar register (a division leaves its result in vector ones).
__device__ __forceinline__ unsigned uniform(unsigned v) { return __builtin_amdgcn_readfirstlane(v); }

struct Place {
  unsigned b, s, c, g;  // sequence, chunk, this lane's channel (clamped into the group), the group
  bool in;              // whether the lane has a channel
};
__device__ __forceinline__ Place place(const Args& a, unsigned id) {
  Place p;
  const unsigned cb = id % a.blocks_c;
  id /= a.blocks_c;
  p.g = id % a.G;
  id /= a.G;
  p.b = uniform(id % (unsigned)a.B);
  p.s = uniform(id / (unsigned)a.B);
  p.g = uniform(p.g);
  const unsigned lc = cb * blockDim.x + threadIdx.x, per = (unsigned)a.per;
  p.in = lc < per;
  p.c = p.g * per + (p.in ? lc : per - 1);
  return p;
}

// B and C of kSteps steps as fp32 in LDS, [Q][step][B, C][4], zero past N and past the sequence's end: loaded to registers
// (get) and later written (put), each thread the values threadIdx.x, + blockDim.x, ... (kMost of them at most). A
// value's place e gives its step (e / 8) % 8, its row (e / 4) % 2 and its state 4 (e / 64) + e % 4.
__device__ __forceinline__ int place_step(int e) { return (e >> 3) & 7; }
__device__ __forceinline__ int place_row(int e) { return (e >> 2) & 1; }
__device__ __forceinline__ int place_state(int e) { return 4 * (e >> 6) + (e & 3); }
static_assert(kSteps == 8, "places of the staged values");
template <typename T, int kMost>
struct StageBC {
  gin<T> p[kMost];     // of step 0
  long stride[kMost];
  int step[kMost];     // of the batch; past it for no value
  T v[kMost];          // as loaded
  __device__ __forceinline__ void init(const Args& a, long b, unsigned g) {
#pragma unroll
    for (int k = 0; k < kMost; k++) {
      const int e = threadIdx.x + k * blockDim.x, n = place_state(e);
      const bool is_c = place_row(e);
      p[k] = is_c ? (gin<T>)a.Cm + b * a.cm_b : (gin<T>)a.Bm + b * a.bm_b;
      p[k] += g * a.N + n;
      stride[k] = is_c ? a.cm_t : a.bm_t;
      step[k] = n < a.N ? place_step(e) : kSteps;
    }
  }
  __device__ __forceinline__ void get(int t0, int steps) {
#pragma unroll
    for (int k = 0; k < kMost; k++) v[k] = step[k] < steps ? p[k][(long)(t0 + step[k]) * stride[k]] : T(0);
  }
  __device__ __forceinline__ void put(const Args& a, float* s) const {
    const int tot = kSteps * 8 * a.Q;
#pragma unroll
    for (int k = 0; k < kMost; k++) {
      const int e = threadIdx.x + k * blockDim.x;
      if (e < tot) s[e] = raw_f32(v[k]);
    }
  }
};

// States n0.. n0 + 3 of a row of N, zero past N.
__device__ __forceinline__ f4t row4(const float* p, int n0, int N) {
  return f4(p[n0], n0 + 1 < N ? p[n0 + 1] : 0.f, n0 + 2 < N ? p[n0 + 2] : 0.f, n0 + 3 < N ? p[n0 + 3] : 0.f);
}
__device__ __forceinline__ void set_row4(float* p, int n0, int N, const f4t& v) {
  p[n0] = v.x;
  if (n0 + 1 < N) p[n0 + 1] = v.y;
  if (n0 + 2 < N) p[n0 + 2] = v.z;
  if (n0 + 3 < N) p[n0 + 3] = v.w;
}
// A in units of the base-2 exponential.
__device__ __forceinline__ f4t decay4(const Args& a, unsigned c, int q) {
  const f4t v = row4(a.A + (long)c * a.N, 4 * q, a.N);
  return f4(v.x * kLog2e, v.y * kLog2e, v.z * kLog2e, v.w * kLog2e);
}

// Raw rows of a batch, loaded a batch ahead; steps past the end repeat the last one. They stay what the load gives, in T:
// anything done to a value where it is loaded, a widening too, would wait for it there.
template <typename T>
struct Rows {
  T v[kSteps];
  __device__ __forceinline__ void get(gin<T> p, long stride, int steps, unsigned c) {
    const Lane<T> at(c);
    if (steps == kSteps) {
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        v[i] = *at(p);
        walk(p, stride);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        v[i] = *at(p);
        walk(p, i + 1 < steps ? stride : 0);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // or the addresses of all rows of a batch are made first
      }
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    return raw_f32(v[i]);
  }
  // From here on the compiler takes the values as new: what is computed from them again is not kept from before.
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int i = 0; i < kSteps; i++) asm("" : "+v"(v[i]));
  }
};

// The window after the last step: its K - 1 inputs, zero where an episode started after them.
template <typename T>
__device__ __forceinline__ void store_window(const Args& a, float* win, long b, unsigned c) {
  const long K1 = a.K - 1;
  float x[kTaps - 1];
  look_back<T>(x, a, a.T, b, c);
  bool same = true;  // no episode has started after the input
#pragma unroll
  for (int j = kTaps - 2; j >= 0; j--) {
    const long k = j - (kTaps - 1 - K1), t = a.T - (kTaps - 1) + j;
    if (k < 0) break;
    win[(b * K1 + k) * a.C + c] = same ? x[j] : 0.f;
    same = same && !starts(a, t, b);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) k_ssm_window(Args a) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i < a.B * a.C) store_window<T>(a, a.win_out, i / a.C, (unsigned)(i % a.C));
}

// A launch of 2^32 threads or more would start the remainder only: its blocks are rows of 2^22 (the last one's excess has no work).
constexpr int kGridRow = 22;
inline dim3 grid_rows(unsigned blocks) {
  return blocks <= 1u << kGridRow ? dim3(blocks) : dim3(1u << kGridRow, (blocks + (1u << kGridRow) - 1) >> kGridRow);
}

// One chunk of one sequence. LOCAL: from a zero state, keeping only the end state and the decay's exponent.
template <typename T, bool LOCAL, int MOST>
__global__ void __launch_bounds__(256) k_ssm_fwd(Args a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int Q = a.Q, nt = blockDim.x, tid = threadIdx.x;
  f4t* sA = reinterpret_cast<f4t*>(lds);  // [Q][nt]
  f4t* sH = sA + Q * nt;                     // [Q][nt]
  float* sbc = lds + 8 * Q * nt;                // [2][Q][kSteps][2][4]
  const Place pl = place(a, (blockIdx.y << kGridRow) + blockIdx.x);
  if (pl.s >= (unsigned)a.chunks) return;
  const long b = pl.b;
  const unsigned c = pl.c;
  const int tbeg = (int)pl.s * a.chunk, tend = min(a.T, tbeg + a.chunk);
  gin<T> xp = (gin<T>)a.x + b * a.x_b + tbeg * a.x_t;
  gin<T> dp = (gin<T>)a.delta + b * a.d_b + tbeg * a.d_t;
  gin<T> zp = (gin<T>)a.z + (a.z ? b * a.z_b + tbeg * a.z_t : 0);
  gout<T> yp = (gout<T>)a.y + b * a.y_b + tbeg * a.y_t;
  const long quads = a.B * Q * a.C;  // quads of the library's states of one chunk (or kept batch)
  gout<f4t> keep = LOCAL || !a.keep ? nullptr : (gout<f4t>)a.keep + tbeg / kSteps * quads + b * Q * a.C;
  Rows<T> rx, rd, rz = {};
  StageBC<T, MOST> bc;
  bc.init(a, b, pl.g);
  float fl, back[kTaps - 1];
  auto fetch = [&](int t0) __attribute__((always_inline)) {
    const int n = min(kSteps, tend - t0);
    bc.get(t0, n);
    rx.get(xp, a.x_t, n, c);
    rd.get(dp, a.d_t, n, c);
    if (!LOCAL && a.z) rz.get(zp, a.z_t, n, c);
    fl = flag_load(a, t0, tend, b);
    walk(xp, kSteps * a.x_t);
    walk(dp, kSteps * a.d_t);
    if (!LOCAL) walk(zp, kSteps * a.z_t);
  };
  fetch(tbeg);
  look_back<T>(back, a, tbeg, b, c);
  Conv cv;
  cv.init(a, c);
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
  for (int q = 0; q < Q; q++) {
    sA[q * nt + tid] = decay4(a, c, q);
    f4t h = f4(0.f, 0.f, 0.f, 0.f);
    if (!LOCAL) {
      if (a.chunks > 1) h = reinterpret_cast<const f4t*>(a.hloc)[pl.s * quads + (b * Q + q) * a.C + c];
      else if (a.h0) h = row4(a.h0 + (b * a.C + c) * a.N, 4 * q, a.N);
    }
    sH[q * nt + tid] = h;
  }
  float dsum = 0.f;
  unsigned cleared = 0;
  int buf = 0;
  for (int t0 = tbeg; t0 < tend; t0 += kSteps, buf ^= 1) {
    // two buffers and one barrier: a wavefront writes this one again only after every wavefront has passed the
    // barrier of the batch between, and so has read it
    float* s = sbc + buf * 64 * Q;
    bc.put(a, s);
    const Rows<T> cx = rx, cd = rd, cz = rz;
    const unsigned bits = flag_bits(fl), st = bits >> (kTaps - 1);
    const int steps = min(kSteps, tend - t0);
    __syncthreads();
    if (t0 + kSteps < tend) fetch(t0 + kSteps);
    cleared |= st;
    float d[kSteps], du[kSteps], o[kSteps];
    // CLEAN: a whole batch that no episode's start cuts, of a convolution of all taps; the other form selects what each step
    // sees. Without a convolution or gate theirs are computed all the same and not taken: a choice per step would split
    // the batch into many short blocks.
    auto prepare = [&](auto CLEAN) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        const int n = decltype(CLEAN)::value ? kTaps - 1 : cv.reach(bits, i);
        const float x1 = i > 0 ? cx[i > 0 ? i - 1 : 0] : back[2], x2 = i > 1 ? cx[i > 1 ? i - 2 : 0] : back[i + 1],
                    x3 = i > 2 ? cx[i > 2 ? i - 3 : 0] : back[i];
        const float w = silu(cv.pre(cx[i], n > 0 ? x1 : 0.f, n > 1 ? x2 : 0.f, n > 2 ? x3 : 0.f));
        const float u = decltype(CLEAN)::value || cv.K ? w : cx[i];
        d[i] = softplus(cd[i] + bias);
        du[i] = d[i] * u;
        if (!decltype(CLEAN)::value) {
          // a step past the end leaves the state as it is: a decay of one and no input
          d[i] = i < steps ? d[i] : 0.f;
          du[i] = i < steps ? du[i] : 0.f;
        }
        if (LOCAL) dsum += d[i];
        o[i] = Dc * u;
      }
    };
    if (bits == 0 && steps == kSteps && cv.K == kTaps) prepare(std::true_type{});
    else prepare(std::false_type{});
#pragma unroll
    for (int j = 0; j < kTaps - 1; j++) back[j] = cx[kSteps - (kTaps - 1) + j];
    auto scan = [&](auto ANY) __attribute__((always_inline)) {  // ANY: an episode starts in this batch
      for (int q = 0; q < Q; q++) {
        const f4t A = sA[q * nt + tid];
        f4t h = sH[q * nt + tid];
        if (!LOCAL && keep && pl.in) *Lane<f4t>(c)(keep + q * a.C) = h;
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
          if constexpr (decltype(ANY)::value) {
            const bool cut = st & (1u << i);
            h = f4(cut ? 0.f : h.x, cut ? 0.f : h.y, cut ? 0.f : h.z, cut ? 0.f : h.w);
          }
          const f4t Bv = *reinterpret_cast<const f4t*>(&s[64 * q + 8 * i]);
          h.x = fmaf(ex2(d[i] * A.x), h.x, du[i] * Bv.x);
          h.y = fmaf(ex2(d[i] * A.y), h.y, du[i] * Bv.y);
          h.z = fmaf(ex2(d[i] * A.z), h.z, du[i] * Bv.z);
          h.w = fmaf(ex2(d[i] * A.w), h.w, du[i] * Bv.w);
          if (!LOCAL) {
            const f4t Cv = *reinterpret_cast<const f4t*>(&s[64 * q + 8 * i + 4]);
            o[i] = fmaf(h.x, Cv.x, fmaf(h.y, Cv.y, fmaf(h.z, Cv.z, fmaf(h.w, Cv.w, o[i]))));
          }
          if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // bounds the values of later steps that are fetched early
        }
        sH[q * nt + tid] = h;
      }
    };
    if (st) scan(std::true_type{});
    else scan(std::false_type{});
    if (!LOCAL) {
      if (keep) walk(keep, quads);
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        const float w = o[i] * silu(cz[i]);
        o[i] = a.z ? w : o[i];
      }
      if (pl.in) {
        if (steps == kSteps) {
          gout<T> p = yp;
          const Lane<T> at(c);
#pragma unroll
          for (int i = 0; i < kSteps; i++) {
            stf(at(p), o[i]);
            walk(p, a.y_t);
          }
        } else {
          for (int i = 0; i < kSteps; i++)
            if (i < steps) stf(yp + i * a.y_t + c, o[i]);
        }
      }
      walk(yp, kSteps * a.y_t);
    }
  }
  if (!pl.in) return;
  for (int q = 0; q < Q; q++) {
    const f4t h = sH[q * nt + tid];
    if (LOCAL) reinterpret_cast<f4t*>(a.hloc)[pl.s * quads + (b * Q + q) * a.C + c] = h;
    else if (tend == a.T && a.h_out) set_row4(a.h_out + (b * a.C + c) * a.N, 4 * q, a.N, h);
  }
  if (LOCAL) a.dsum[(pl.s * a.B + b) * a.C + c] = cleared ? -1.f : dsum;
  else if (tend == a.T && a.win_here) store_window<T>(a, a.win_out, b, c);
}

// A thread's state in the library's layout, [B][Q][C][4].
struct StateAt {
  long bc, c, n;
  bool in;
};
__device__ __forceinline__ StateAt state_at(const Args& a, long i) {
  const long c = i / 4 % a.C, q = i / (4 * a.C) % a.Q, b = i / (4 * a.C * a.Q), n = 4 * q + i % 4;
  return {b * a.C + c, c, n, n < a.N};
}
// run -> decay run + local over the chunks in order, each chunk's entry replaced by the run before it. A chain of short
// steps, so the loads of sixteen of them go ahead of it.
template <int DIR>
__device__ __forceinline__ void join(float* loc, long row, const float* dsum, long drow, int chunks, float A2, float run) {
  constexpr int kAhead = 16;
  for (int s0 = 0; s0 < chunks; s0 += kAhead) {
    float l[kAhead], d[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const long s = min(s0 + k, chunks - 1);
      l[k] = loc[DIR * s * row];
      d[k] = dsum[DIR * s * drow];
    }
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      if (s0 + k >= chunks) break;
      loc[DIR * (long)(s0 + k) * row] = run;
      run = d[k] < 0.f ? l[k] : fmaf(ex2(A2 * d[k]), run, l[k]);
    }
  }
}

// Joins the chunks in order: hloc[s] becomes the state before chunk s. One thread per state.
__global__ void __launch_bounds__(256) k_ssm_join(Args a) {
  const long row = a.B * a.C * 4 * a.Q, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= row) return;
  const StateAt at = state_at(a, i);
  const float A2 = at.in ? a.A[at.c * a.N + at.n] * kLog2e : 0.f;
  join<1>(a.hloc + i, row, a.dsum + at.bc, a.B * a.C, a.chunks, A2, at.in && a.h0 ? a.h0[at.bc * a.N + at.n] : 0.f);
}

// ---- single tokens -------------------------------------------------------------------------------------
// Four consecutive elements of a row of B or C.
__device__ __forceinline__ f4t quad_of(const float* p) { return *reinterpret_cast<const f4t*>(p); }
__device__ __forceinline__ f4t quad_of(const uint16_t* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return f4(__builtin_bit_cast(float, v.x << 16), __builtin_bit_cast(float, v.x & 0xffff0000u),
                     __builtin_bit_cast(float, v.y << 16), __builtin_bit_cast(float, v.y & 0xffff0000u));
}

// One step of every sequence, the state updated in place: bound by the state's 8 bytes per element, so what a channel
// needs once (convolution, time step, gate) is computed once, by the lane of that channel, and handed over through LDS to
// the lanes that move the state, each four states of it as one 16-byte access (consecutive lanes, consecutive
// addresses). Measured, 4096 x 512 channels of 16 states: 82 us, 4.1 TB/s; a large copy would take 68. QT: Q where it is 1, 2 or
// 4 and every access may be a vector one, with the decays in registers over the block's sequences; 0: any Q, in single
// elements (4, 8 and 16 states 29, 52 and 78 us against 45, 91 and 157; the states that have no other form: 12 132, 24 236, 32
// 304, 64 582, at 2 TB/s).
template <typename T, int QT>
__global__ void __launch_bounds__(256) k_ssm_step(Args a, float* __restrict__ hs, float* __restrict__ win, int per_block) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int nt = blockDim.x, tid = threadIdx.x, Q = QT ? QT : a.Q, N = a.N;
  float* sd = lds;           // [nt] d
  float* sdu = lds + nt;     // [nt] d u
  float* so = lds + 2 * nt;  // [nt][Q] shares of <h, C>
  const unsigned nblk = (unsigned)((a.C + nt - 1) / nt), cb = uniform(blockIdx.x % nblk);
  const long b0 = (long)uniform(blockIdx.x / nblk) * per_block, b1 = min(a.B, b0 + per_block);
  const long c0 = (long)cb * nt;
  const bool in = c0 + tid < a.C;
  const unsigned c = (unsigned)(in ? c0 + tid : a.C - 1);
  const int K = a.K, chans = (int)min((long)nt, a.C - c0);
  Conv cv;
  cv.init(a, c);
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
  f4t Av[QT ? QT : 1];
  int lcs[QT ? QT : 1], goff[QT ? QT : 1];
  if constexpr (QT > 0) {
#pragma unroll
    for (int j = 0; j < QT; j++) {
      const int idx = j * nt + tid, lc = idx / QT;
      lcs[j] = lc;
      const long ch = c0 + (lc < chans ? lc : 0);
      goff[j] = (int)(ch / a.per) * N + 4 * (idx % QT);
      const f4t v = lc < chans ? *reinterpret_cast<const f4t*>(a.A + c0 * N + 4 * idx) : f4(0.f, 0.f, 0.f, 0.f);
      Av[j] = f4(v.x * kLog2e, v.y * kLog2e, v.z * kLog2e, v.w * kLog2e);
    }
  }
  for (long b = b0; b < b1; b++) {
    const bool clear = a.first && a.first[b] != 0.f;
    float* hb = hs + (b * a.C + c0) * N;
    const T* Bp = (const T*)a.Bm + b * a.bm_b;
    const T* Cp = (const T*)a.Cm + b * a.cm_b;
    f4t hv[QT ? QT : 1];
    if constexpr (QT > 0) {  // the state's loads first
#pragma unroll
      for (int j = 0; j < QT; j++)
        hv[j] = lcs[j] < chans && !clear ? *reinterpret_cast<const f4t*>(hb + 4 * (j * nt + tid)) : f4(0.f, 0.f, 0.f, 0.f);
    }
    const float x = ldf((gin<T>)a.x + b * a.x_b + c);
    float u = x;
    if (K) {
      float* wp = win + b * (K - 1) * a.C;
      const float x1 = K > 1 && !clear ? wp[(K - 2) * a.C + c] : 0.f, x2 = K > 2 && !clear ? wp[(K - 3) * a.C + c] : 0.f,
                  x3 = K > 3 && !clear ? wp[c] : 0.f;
      u = silu(cv.pre(x, x1, x2, x3));
      if (in) {  // the window moves on
        if (K > 1) wp[(K - 2) * a.C + c] = x;
        if (K > 2) wp[(K - 3) * a.C + c] = x1;
        if (K > 3) wp[c] = x2;
      }
    }
    const float d = softplus(ldf((gin<T>)a.delta + b * a.d_b + c) + bias);
    sd[tid] = d;
    sdu[tid] = d * u;
    __syncthreads();
    if constexpr (QT > 0) {
#pragma unroll
      for (int j = 0; j < QT; j++) {
        if (lcs[j] >= chans) continue;
        const float dd = sd[lcs[j]], du = sdu[lcs[j]];
        const f4t Bv = quad_of(Bp + goff[j]), Cv = quad_of(Cp + goff[j]), A = Av[j];
        f4t h = hv[j];
        h.x = fmaf(ex2(dd * A.x), h.x, du * Bv.x);
        h.y = fmaf(ex2(dd * A.y), h.y, du * Bv.y);
        h.z = fmaf(ex2(dd * A.z), h.z, du * Bv.z);
        h.w = fmaf(ex2(dd * A.w), h.w, du * Bv.w);
        *reinterpret_cast<f4t*>(hb + 4 * (j * nt + tid)) = h;
        so[j * nt + tid] = fmaf(h.x, Cv.x, fmaf(h.y, Cv.y, fmaf(h.z, Cv.z, h.w * Cv.w)));
      }
    } else {
      for (int idx = tid; idx < chans * Q; idx += nt) {
        const int lc = idx / Q, n0 = 4 * (idx - lc * Q);
        const long ch = c0 + lc, g = ch / a.per;
        const float dd = sd[lc], du = sdu[lc];
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int n = n0 + i;
          if (n >= N) break;
          float h = clear ? 0.f : hb[lc * N + n];
          h = fmaf(ex2(dd * (a.A[ch * N + n] * kLog2e)), h, du * ldf(Bp + g * N + n));
          hb[lc * N + n] = h;
          o = fmaf(h, ldf(Cp + g * N + n), o);
        }
        so[idx] = o;
      }
    }
    __syncthreads();
    if (in) {
      float o = Dc * u;
      for (int q = 0; q < Q; q++) o += so[tid * Q + q];
      if (a.z) o *= silu(ldf((gin<T>)a.z + b * a.z_b + c));
      stf((gout<T>)a.y + b * a.y_b + c, o);
    }
    // the next sequence writes sd and sdu, which nobody reads any more, and so only after its own barrier
  }
}

// ---- gradient ------------------------------------------------------------------------------------------
struct GradArgs {
  const void* dy;
  long dy_t, dy_b;
  void *dx, *dz, *ddelta, *dB, *dC;
  long dx_t, dx_b, dz_t, dz_b, dd_t, dd_b, db_t, db_b, dc_t, dc_b;
  const float* keep;
  float* carry;   // [chunks] states: each chunk's own adjoint at its start, then the one coming in at its end
  float* bc;      // [blocks_c][T][B][G][2][N] sums of dB, dC over a block's channels
  float* par;     // [rows][C][P] sums of the parameters' gradients over a block's work, P = N + K + 3
  float* halo;    // [chunks][B][K-1][C]: what a chunk adds to dx of the K - 1 steps before it
  long rows;      // blocks that share a channel block's work
  int P;
};

// Sums over the 64 lanes of eight values at each of eight steps, in two halves. lane_sums takes a step's eight values and
// leaves in lane l a partial of value l / 8, over the lanes of the same l % 8: two values at a time are folded by swapping
// wavefront halves, then rows of 16 lanes, then lanes eight apart. step_sums takes the eight steps' partials and
// leaves in lane l the total of value l / 8 at step l % 8. Together under 20 instructions a step, where eight
// separate sums would take 48.
template <int CTL> __device__ __forceinline__ float fold_dpp(float lo, float hi, bool up) {
  return (up ? hi : lo) + dpp_mov<CTL>(up ? lo : hi);
}
__device__ __forceinline__ float lane_sums(float (&v)[8], int lane) {
  swap32(v[0], v[4], v[1], v[5]);
  swap32(v[2], v[6], v[3], v[7]);
  float a = v[0] + v[4], b = v[1] + v[5], c = v[2] + v[6], d = v[3] + v[7];  // values k (lower half) and k + 4
  swap16(a, c, b, d);
  a += c;  // value 4 bit5 + 2 bit4
  b += d;  // the one after it
  return fold_dpp<0x128>(a, b, lane & 8);  // lane ^ 8
}
__device__ __forceinline__ float step_sums(const float (&p)[8], int lane) {
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = fold_dpp<0x141>(p[i], p[i + 4], lane & 4);  // lane ^ 7
  const float a = fold_dpp<0x4E>(r[0], r[2], lane & 2), b = fold_dpp<0x4E>(r[1], r[3], lane & 2);  // lane ^ 2
  return fold_dpp<0xB1>(a, b, lane & 1);  // lane ^ 1
}

// The adjoint that a chunk alone sends back past its first step (its own outputs only).
template <typename T, int MOST>
__global__ void __launch_bounds__(256) k_ssm_bwd_local(Args a, GradArgs ga) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int Q = a.Q, nt = blockDim.x, tid = threadIdx.x;
  f4t* sA = reinterpret_cast<f4t*>(lds);  // [Q][nt]
  f4t* sG = sA + Q * nt;                     // [Q][nt]
  float* sbc = lds + 8 * Q * nt;                // [2][Q][kSteps][2][4]
  const Place pl = place(a, blockIdx.x);
  const long b = pl.b;
  const unsigned c = pl.c;
  const int tbeg = (int)pl.s * a.chunk, tend = min(a.T, tbeg + a.chunk);
  const int tlast = tbeg + (tend - tbeg - 1) / kSteps * kSteps;
  for (int q = 0; q < Q; q++) {
    sA[q * nt + tid] = decay4(a, c, q);
    sG[q * nt + tid] = f4(0.f, 0.f, 0.f, 0.f);
  }
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.f;
  float dsum = 0.f;
  unsigned cleared = 0;
  Rows<T> rd, rz = {}, rg;
  StageBC<T, MOST> bc;
  bc.init(a, b, pl.g);
  float fl;
  auto fetch = [&](int t0) __attribute__((always_inline)) {
    const int n = min(kSteps, tend - t0);
    bc.get(t0, n);
    rd.get((gin<T>)a.delta + b * a.d_b + t0 * a.d_t, a.d_t, n, c);
    if (a.z) rz.get((gin<T>)a.z + b * a.z_b + t0 * a.z_t, a.z_t, n, c);
    rg.get((gin<T>)ga.dy + b * ga.dy_b + t0 * ga.dy_t, ga.dy_t, n, c);
    fl = flag_load(a, t0, tend, b);
  };
  fetch(tlast);
  int buf = 0;
  for (int t0 = tlast; t0 >= tbeg; t0 -= kSteps, buf ^= 1) {
    float* s = sbc + buf * 64 * Q;
    bc.put(a, s);
    const Rows<T> cd = rd, cz = rz, cg = rg;
    const unsigned st = flag_bits(fl) >> (kTaps - 1);
    const int steps = min(kSteps, tend - t0);
    __syncthreads();
    if (t0 > tbeg) fetch(t0 - kSteps);
    cleared |= st;
    float d[kSteps], dout[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      d[i] = i < steps ? softplus(cd[i] + bias) : 0.f;
      dout[i] = i < steps ? (a.z ? cg[i] * silu(cz[i]) : cg[i]) : 0.f;
      dsum += d[i];
    }
    for (int q = 0; q < Q; q++) {
      const f4t A = sA[q * nt + tid];
      f4t g = sG[q * nt + tid];
#pragma unroll
      for (int i = kSteps - 1; i >= 0; i--) {
        const f4t Cv = *reinterpret_cast<const f4t*>(&s[64 * q + 8 * i + 4]);
        g.x = ex2(d[i] * A.x) * fmaf(dout[i], Cv.x, g.x);
        g.y = ex2(d[i] * A.y) * fmaf(dout[i], Cv.y, g.y);
        g.z = ex2(d[i] * A.z) * fmaf(dout[i], Cv.z, g.z);
        g.w = ex2(d[i] * A.w) * fmaf(dout[i], Cv.w, g.w);
        if (st & (1u << i)) g = f4(0.f, 0.f, 0.f, 0.f);
      }
      sG[q * nt + tid] = g;
    }
  }
  if (!pl.in) return;
  gout<f4t> out = (gout<f4t>)ga.carry + (pl.s * a.B + b) * Q * a.C + c;
  for (int q = 0; q < Q; q++) out[q * a.C] = sG[q * nt + tid];
  a.dsum[(pl.s * a.B + b) * a.C + c] = cleared ? -1.f : dsum;
}

// Joins them from the end: carry[s] becomes the adjoint that comes in at chunk s's last step.
__global__ void __launch_bounds__(256) k_ssm_bwd_join(Args a, GradArgs ga) {
  const long row = a.B * a.C * 4 * a.Q, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= row) return;
  const StateAt at = state_at(a, i);
  const float A2 = at.in ? a.A[at.c * a.N + at.n] * kLog2e : 0.f;
  const long last = a.chunks - 1;
  join<-1>(ga.carry + last * row + i, row, a.dsum + last * a.B * a.C + at.bc, a.B * a.C, a.chunks, A2, 0.f);
}

// The gradient of one chunk after another. Batches of kSteps steps run backwards in time. Each takes the states four at
// a time: from the kept states it runs its steps forward again, keeping the decay a_t and a_t h_{t-1} of every step
// in registers (64 of them), then runs them backwards, g_t = C_t dout_t + a_{t+1} g_{t+1}. So the decays are computed once
// per batch and two wavefronts share a SIMD; the other states' A, g and dA rest in the lane's LDS slots.
//
// With q = g a_t h_{t-1} per state: dA += d q, d(d) = sum A q + u sum g B, du = d sum g B, dB = sum_c g d u, dC = sum_c
// h dout. The two sums over channels take g and a_t h_{t-1} as they are and add the step's own share, C_n or B_n times
// S = sum_c dout d u, where they are joined; the sums over states likewise add dout (or d u) times <B, C>, which
// the staging computes once per step. Sums over channels are folded over the wavefront's lanes, then over the
// block's wavefronts in LDS; the parameters' gradients stay in LDS and registers over all the block's work. A block
// takes the items row, row + rows, ... of its channel block, an item being a chunk of a sequence.
constexpr int kOwn = 3 + kTaps;  // a channel's own sums in the gradient
static_assert(kOwn == kSsmOwn, "LDS of a block");
template <typename T, int MOST>
__global__ void __launch_bounds__(256, 2) k_ssm_bwd(Args a, GradArgs ga) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int Q = a.Q, nt = blockDim.x, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, waves = nt >> 6;
  f4t* sA = reinterpret_cast<f4t*>(lds);  // [Q][nt]
  f4t* sG = sA + Q * nt;                     // [Q][nt]
  f4t* sdA = sG + Q * nt;                    // [Q][nt]
  float* sbc = lds + 12 * Q * nt;               // [2][Q][kSteps][B, C][4]
  float* red = sbc + 2 * 64 * Q;                // [waves][Q][kSteps][dB, dC][4]
  float* reds = red + waves * 64 * Q;           // [waves][kSteps] of S
  float* scb = reds + waves * kSteps;           // [2][kSteps] of <B, C>
  float* own = scb + 2 * kSteps;                // [kOwn][nt]: dD, d(dt_bias), d(conv_b), d(conv_w)
  const unsigned cb = uniform(blockIdx.x % a.blocks_c), grp = uniform((blockIdx.x / a.blocks_c) % a.G);
  const unsigned row = uniform(blockIdx.x / (a.blocks_c * a.G)), items = (unsigned)(a.B * a.chunks);
  const unsigned lc = cb * nt + tid;
  const bool in = lc < (unsigned)a.per;
  const unsigned c = grp * (unsigned)a.per + (in ? lc : (unsigned)a.per - 1);
  const int out = 8 * (lane & 7) + (lane >> 3);  // place of the total that step_sums leaves in this lane
  Conv cv;
  cv.init(a, c);
  for (int q = 0; q < Q; q++) {
    sA[q * nt + tid] = decay4(a, c, q);
    sdA[q * nt + tid] = f4(0.f, 0.f, 0.f, 0.f);
  }
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
#pragma unroll
  for (int k = 0; k < kOwn; k++) own[k * nt + tid] = 0.f;
  const int K = cv.K;
  const long quads = a.B * Q * a.C;
  // What a batch reads: the rows, the three inputs before them, the flags, the first kept states and this thread's share of B
  // and C, as loaded. The next batch's are on their way while a batch computes its channels' own gradients, where the
  // registers of the states' steps are free again.
  struct Where {
    unsigned b, s;
    int tbeg, tend, t0;
  };
  auto enter = [&](unsigned item) __attribute__((always_inline)) {  // the last batch of an item
    Where w;
    w.b = uniform(item % (unsigned)a.B);
    w.s = uniform(item / (unsigned)a.B);
    w.tbeg = (int)w.s * a.chunk;
    w.tend = min(a.T, w.tbeg + a.chunk);
    w.t0 = w.tbeg + (w.tend - w.tbeg - 1) / kSteps * kSteps;
    return w;
  };
  Rows<T> rx, rd, rz = {}, rg;
  T before[kTaps - 1] = {}, vbc[MOST];
  float fl;
  f4t next;
  auto fetch = [&](const Where& w) __attribute__((always_inline)) {
    const Args a = again<Args>(0);
    const GradArgs ga = again<GradArgs>(sizeof(Args));
    const long b = w.b;
    const int t0 = w.t0, steps = min(kSteps, w.tend - t0);
    rx.get((gin<T>)a.x + b * a.x_b + t0 * a.x_t, a.x_t, steps, c);
    if (t0 > 0) {
      gin<T> p = (gin<T>)a.x + b * a.x_b + (t0 - (kTaps - 1)) * a.x_t;
      const Lane<T> at(c);
#pragma unroll
      for (int j = 0; j < kTaps - 1; j++) {
        before[j] = *at(p);
        walk(p, a.x_t);
      }
    }
    rd.get((gin<T>)a.delta + b * a.d_b + t0 * a.d_t, a.d_t, steps, c);
    if (a.z) rz.get((gin<T>)a.z + b * a.z_b + t0 * a.z_t, a.z_t, steps, c);
    rg.get((gin<T>)ga.dy + b * ga.dy_b + t0 * ga.dy_t, ga.dy_t, steps, c);
    next = *Lane<f4t>(c)((gin<f4t>)ga.keep + t0 / kSteps * quads + b * Q * a.C);
    int me = tid;
    asm("" : "+v"(me));  // or the places of all MOST values wait in registers over the states' steps
#pragma unroll
    for (int k = 0; k < MOST; k++) {
      const int e = me + k * nt, n = place_state(e), i = place_step(e);
      const bool is_c = place_row(e);
      gin<T> p = is_c ? (gin<T>)a.Cm + b * a.cm_b : (gin<T>)a.Bm + b * a.bm_b;
      vbc[k] = n < a.N && i < steps ? p[(long)(t0 + i) * (is_c ? a.cm_t : a.bm_t) + grp * a.N + n] : T(0);
    }
    fl = flag_load(a, t0, w.tend, b);
  };
  int buf = 0;
  unsigned item = row;
  if (item >= items) return;  // (a block without work: the launch has none)
  Where at = enter(item);
  fetch(at);
  // ds of the three steps after the current one, of the same episode (zero past the chunk: its successor's
  // share of this chunk's last steps comes through the halo)
  float q1 = 0.f, q2 = 0.f, q3 = 0.f;
  for (;; buf ^= 1) {
    const long b = at.b, s = at.s;
    const int tbeg = at.tbeg, tend = at.tend, t0 = at.t0;
    if (t0 + kSteps >= tend) {
      q1 = q2 = q3 = 0.f;
      gin<f4t> carry = (gin<f4t>)ga.carry + s * quads + b * Q * a.C;
      for (int q = 0; q < Q; q++)  // a lane without a channel sends nothing back, and so adds nothing to a sum
        sG[q * nt + tid] = a.chunks > 1 && in ? (carry + q * a.C)[c] : f4(0.f, 0.f, 0.f, 0.f);
    }
    Where to = at;  // the batch after this one
    to.t0 = t0 - kSteps;
    bool more = true;
    if (t0 == tbeg) {
      item += (unsigned)ga.rows;
      more = item < items;
      if (more) to = enter(item);
    }
    {
      const int steps = min(kSteps, tend - t0);
      gin<f4t> keep = (gin<f4t>)ga.keep + t0 / kSteps * quads + b * Q * a.C;
      Rows<T> cx = rx, cd = rd, cz = rz, cg = rg;
      float back[kTaps - 1];
      if (t0 > 0) {
#pragma unroll
        for (int j = 0; j < kTaps - 1; j++) back[j] = raw_f32(before[j]);
      } else {
        look_back<T>(back, a, 0, b, c);
      }
      const unsigned bits = flag_bits(fl), st = bits >> (kTaps - 1);
      float* sb = sbc + buf * 64 * Q;
#pragma unroll
      for (int k = 0; k < MOST; k++)
        if (tid + k * nt < 64 * Q) sb[tid + k * nt] = raw_f32(vbc[k]);
      // Input j (0..10) of the batch and of the three steps before it, and a step's own convolution. CLEAN as in the forward.
      auto input = [&](int j) __attribute__((always_inline)) { return j < kTaps - 1 ? back[j < kTaps - 1 ? j : 0] : cx[j < kTaps - 1 ? 0 : j - (kTaps - 1)]; };
      auto conv = [&](auto CLEAN, int i, float& x1, float& x2, float& x3) __attribute__((always_inline)) {
        const int n = decltype(CLEAN)::value ? kTaps - 1 : cv.reach(bits, i);
        x1 = n > 0 ? input(i + 2) : 0.f;
        x2 = n > 1 ? input(i + 1) : 0.f;
        x3 = n > 2 ? input(i) : 0.f;
        return cv.pre(cx[i], x1, x2, x3);
      };
      const bool clean = bits == 0 && steps == kSteps && K == kTaps;
      float d[kSteps], du[kSteps], dout[kSteps], o[kSteps], gB[kSteps], Aq[kSteps];
      auto prepare = [&](auto CLEAN) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
          float x1, x2, x3;
          const float w = silu(conv(CLEAN, i, x1, x2, x3)), u = decltype(CLEAN)::value || K ? w : cx[i], gated = cg[i] * silu(cz[i]);
          d[i] = softplus(cd[i] + bias);
          du[i] = d[i] * u;
          dout[i] = a.z ? gated : cg[i];
          if (!decltype(CLEAN)::value) {
            // a step past the end neither decays, nor takes nor gives
            d[i] = i < steps ? d[i] : 0.f;
            du[i] = i < steps ? du[i] : 0.f;
            dout[i] = i < steps ? dout[i] : 0.f;
          }
          dout[i] = in ? dout[i] : 0.f;
          o[i] = gB[i] = Aq[i] = 0.f;
        }
      };
      if (clean) prepare(std::true_type{});
      else prepare(std::false_type{});
      __syncthreads();
      if (tid < kSteps) {  // read after the barrier below
        float p = 0.f;
        for (int q = 0; q < Q; q++)
          for (int n = 0; n < 4; n++) p = fmaf(sb[64 * q + 8 * tid + n], sb[64 * q + 8 * tid + 4 + n], p);
        scb[buf * kSteps + tid] = p;
      }
      auto scan = [&](auto ANY) __attribute__((always_inline)) {  // ANY: an episode starts in this batch
        for (int q = 0; q < Q; q++) {
          const f4t A = sA[q * nt + tid], kh = next;
          next = *Lane<f4t>(c)(keep + (q + 1 < Q ? q + 1 : q) * a.C);
          const f4t g4 = sG[q * nt + tid];
          const float Av[4] = {A.x, A.y, A.z, A.w};
          float h[4] = {kh.x, kh.y, kh.z, kh.w}, g[4] = {g4.x, g4.y, g4.z, g4.w}, dA[4] = {};
          float dec[kSteps][4], ah[kSteps][4], part[kSteps];
#pragma unroll
          for (int i = 0; i < kSteps; i++) {
            const bool cut = decltype(ANY)::value && (st & (1u << i));
            const f4t Bv = *reinterpret_cast<const f4t*>(&sb[64 * q + 8 * i]);
            const float Bn[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
#pragma unroll
            for (int n = 0; n < 4; n++) {
              dec[i][n] = ex2(d[i] * Av[n]);
              ah[i][n] = dec[i][n] * (cut ? 0.f : h[n]);
              h[n] = fmaf(du[i], Bn[n], ah[i][n]);
            }
            if (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // bounds the values of later steps that are fetched early
          }
#pragma unroll
          for (int i = kSteps - 1; i >= 0; i--) {
            const bool cut = decltype(ANY)::value && (st & (1u << i));
            const f4t Bv = *reinterpret_cast<const f4t*>(&sb[64 * q + 8 * i]);
            const f4t Cv = *reinterpret_cast<const f4t*>(&sb[64 * q + 8 * i + 4]);
            const float Bn[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, Cn[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
            float v[8];
#pragma unroll
            for (int n = 0; n < 4; n++) {
              v[n] = g[n] * du[i];
              v[4 + n] = ah[i][n] * dout[i];
              gB[i] = fmaf(g[n], Bn[n], gB[i]);
              o[i] = fmaf(ah[i][n], Cn[n], o[i]);
              const float gn = fmaf(dout[i], Cn[n], g[n]), qn = gn * ah[i][n];
              Aq[i] = fmaf(Av[n], qn, Aq[i]);
              dA[n] = fmaf(d[i], qn, dA[n]);
              g[n] = cut ? 0.f : dec[i][n] * gn;
            }
            part[i] = lane_sums(v, lane);
            __builtin_amdgcn_sched_barrier(0);
          }
          red[(wave * Q + q) * 64 + out] = step_sums(part, lane);
          sG[q * nt + tid] = f4(g[0], g[1], g[2], g[3]);
          const f4t acc = sdA[q * nt + tid];
          sdA[q * nt + tid] = f4(acc.x + dA[0], acc.y + dA[1], acc.z + dA[2], acc.w + dA[3]);
        }
      };
      if (st) scan(std::true_type{});
      else scan(std::false_type{});
      {
        float v[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; i++) v[i] = dout[i] * du[i];
        float S = lane_sums(v, lane);  // of step lane / 8, over lanes of the same lane % 8
        S += dpp_mov<0x141>(S);
        S += dpp_mov<0x4E>(S);
        S += dpp_mov<0xB1>(S);
        if ((lane & 7) == 0) reds[wave * kSteps + (lane >> 3)] = S;
      }
      __syncthreads();
      if (more) fetch(to);
      const Args aa = again<Args>(0);
      const GradArgs gg = again<GradArgs>(sizeof(Args));
      // the block's sums over its wavefronts, in order
      for (int e = tid; e < 64 * Q; e += nt) {
        const int i = place_step(e), which = place_row(e), n = place_state(e);
        if (n >= aa.N || i >= steps) continue;
        float sum = 0.f, S = 0.f;
        for (int w = 0; w < waves; w++) {
          sum += red[w * 64 * Q + e];
          S += reds[w * kSteps + i];
        }
        sum = fmaf(sb[e ^ 4], S, sum);
        const long t = t0 + i;
        if (gg.bc) gg.bc[((((long)cb * aa.T + t) * aa.B + b) * aa.G + grp) * 2 * aa.N + which * aa.N + n] = sum;
        else if (which && gg.dC) stf((gout<T>)gg.dC + t * gg.dc_t + b * gg.dc_b + grp * aa.N + n, sum);
        else if (!which && gg.dB) stf((gout<T>)gg.dB + t * gg.db_t + b * gg.db_b + grp * aa.N + n, sum);
      }
      // the channel's own gradients
      cx.renew();
      cd.renew();
      cz.renew();
      const int last = t0 + steps - 1;
      float cb2[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; i++) cb2[i] = scb[buf * kSteps + i];
      float dxv[kSteps], ddt[kSteps], dzv[kSteps];
      float dD = own[tid], dbias = own[nt + tid], dcb = own[2 * nt + tid], dw[kTaps];
#pragma unroll
      for (int k = 0; k < kTaps; k++) dw[k] = own[(3 + k) * nt + tid];
      auto finish = [&](auto CLEAN, auto WHOLE) __attribute__((always_inline)) {  // WHOLE: no step is past the end
#pragma unroll
        for (int i = kSteps - 1; i >= 0; i--) {
          if (!decltype(WHOLE)::value && i >= steps) continue;
          float x1, x2, x3;
          const float pre = conv(CLEAN, i, x1, x2, x3), sg = sigma(pre), w = pre * sg, u = decltype(CLEAN)::value || K ? w : cx[i];
          const float gb = fmaf(dout[i], cb2[i], gB[i]);
          ddt[i] = fmaf(u, gb, Aq[i] * (1.f / kLog2e)) * sigma(cd[i] + bias);
          dzv[i] = cg[i] * fmaf(du[i], cb2[i], fmaf(Dc, u, o[i])) * dsilu(cz[i], sigma(cz[i]));
          const float dus = fmaf(d[i], gb, Dc * dout[i]), ds = dus * dsilu(pre, sg);
          dD = fmaf(dout[i], u, dD);
          dbias += ddt[i];
          dcb += ds;
          dw[3] = fmaf(ds, cx[i], dw[3]);
          dw[2] = fmaf(ds, x1, dw[2]);
          dw[1] = fmaf(ds, x2, dw[1]);
          dw[0] = fmaf(ds, x3, dw[0]);
          const float dc = fmaf(cv.w[3], ds, fmaf(cv.w[2], q1, fmaf(cv.w[1], q2, cv.w[0] * q3)));
          dxv[i] = decltype(CLEAN)::value || K ? dc : dus;
          const bool cut = !decltype(CLEAN)::value && (st & (1u << i));
          q3 = cut || (!decltype(CLEAN)::value && K < 4) ? 0.f : q2;
          q2 = cut || (!decltype(CLEAN)::value && K < 3) ? 0.f : q1;
          q1 = cut || (!decltype(CLEAN)::value && K < 2) ? 0.f : ds;
        }
      };
      if (clean) finish(std::true_type{}, std::true_type{});
      else if (steps == kSteps) finish(std::false_type{}, std::true_type{});
      else finish(std::false_type{}, std::false_type{});
      own[tid] = dD;
      own[nt + tid] = dbias;
      own[2 * nt + tid] = dcb;
#pragma unroll
      for (int k = 0; k < kTaps; k++) own[(3 + k) * nt + tid] = dw[k];
      if (in) {
        // the last K - 1 steps of a chunk that has a successor are finished by the halo's launch
        const bool halo = tend < aa.T && t0 + kSteps >= tend && K > 1;
        if (steps == kSteps && !halo && gg.ddelta && gg.dx) {
          gout<T> pd = (gout<T>)gg.ddelta + b * gg.dd_b + t0 * gg.dd_t;
          gout<T> px = (gout<T>)gg.dx + b * gg.dx_b + t0 * gg.dx_t;
          const Lane<T> at(c);
#pragma unroll
          for (int i = 0; i < kSteps; i++) {
            stf(at(pd), ddt[i]);
            stf(at(px), dxv[i]);
            walk(pd, gg.dd_t);
            walk(px, gg.dx_t);
          }
          if (gg.dz) {
            gout<T> pz = (gout<T>)gg.dz + b * gg.dz_b + t0 * gg.dz_t;
#pragma unroll
            for (int i = 0; i < kSteps; i++) {
              stf(at(pz), dzv[i]);
              walk(pz, gg.dz_t);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < kSteps; i++) {
            if (i >= steps) break;
            const int t = t0 + i;
            if (gg.ddelta) stf((gout<T>)gg.ddelta + b * gg.dd_b + t * gg.dd_t + c, ddt[i]);
            if (gg.dz) stf((gout<T>)gg.dz + b * gg.dz_b + t * gg.dz_t + c, dzv[i]);
            if (gg.dx) {
              if (!halo || last - t >= K - 1) stf((gout<T>)gg.dx + b * gg.dx_b + t * gg.dx_t + c, dxv[i]);
              else ((gout<float>)gg.halo + ((s * 2 * aa.B + b) * (kTaps - 1) + (last - t)) * aa.C)[c] = dxv[i];
            }
          }
        }
      }
    }
    // what this chunk adds to dx of the K - 1 steps before it: step tbeg - 1 - j takes ds of up to K - 1 - j steps on
    if (t0 == tbeg && in && K > 1 && s > 0 && ga.dx) {
      const float hq[kTaps - 1] = {fmaf(cv.w[2], q1, fmaf(cv.w[1], q2, cv.w[0] * q3)), fmaf(cv.w[1], q1, cv.w[0] * q2),
                                   cv.w[0] * q1};
#pragma unroll
      for (int j = 0; j < kTaps - 1; j++)
        if (j < K - 1) ga.halo[(((s * 2 - 1) * a.B + b) * (kTaps - 1) + j) * a.C + c] = hq[j];
    }
    if (!more) break;
    at = to;
  }
  if (in && ga.par) {
    float* p = ga.par + ((long)row * a.C + c) * ga.P;
    for (int q = 0; q < Q; q++) set_row4(p, 4 * q, a.N, sdA[q * nt + tid]);
    p += a.N;
    p[0] = own[tid];
    p[1] = own[nt + tid];
    p[2] = K ? own[2 * nt + tid] : 0.f;  // without taps there is no convolution for a bias to be of: u is x
#pragma unroll
    for (int k = 0; k < kTaps; k++)
      if (k >= kTaps - K) p[3 + k - (kTaps - K)] = own[(3 + k) * nt + tid];
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
  stf((gout<T>)ga.dx + t * ga.dx_t + b * ga.dx_b + c, v);
}

// dB, dC = the channel blocks' sums in order.
template <typename T>
__global__ void __launch_bounds__(256) k_ssm_fold_bc(Args a, GradArgs ga) {
  const long G = a.G, W = G * 2 * a.N, tot = a.T * a.B * W;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < tot; i += (long)gridDim.x * 256) {
    const long tb = i / W, b = tb % a.B, t = tb / a.B;
    const long e = i % W, g = e / (2 * a.N), r = e % (2 * a.N), which = r / a.N, n = r % a.N;
    float s = 0.f;
    for (int cb = 0; cb < a.blocks_c; cb++) s += ga.bc[cb * tot + i];
    if (which) {
      if (ga.dC) stf((gout<T>)ga.dC + t * ga.dc_t + b * ga.dc_b + g * a.N + n, s);
    } else if (ga.dB) {
      stf((gout<T>)ga.dB + t * ga.db_t + b * ga.db_b + g * a.N + n, s);
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
  const long per = (rows + 3) / 4, end = min(rows, (z + 1) * per);
  for (long i0 = (long)blockIdx.x * 64; i0 < CP; i0 += (long)gridDim.x * 64) {
    const long i = i0 + e;
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
    __syncthreads();  // the sums before have been read
    sh[z][e] = s;
    __syncthreads();
    if (z || i >= CP) continue;
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
  a.T = (int)p.T; a.B = (long)p.B; a.C = (int)p.C; a.N = (int)p.N; a.per = (int)(p.C / p.G); a.K = (int)p.K;
  a.G = (unsigned)p.G;
  a.Q = (int)((p.N + 3) / 4);
  a.x = p.x; a.z = p.z; a.delta = p.delta; a.Bm = p.Bm; a.Cm = p.Cm;
  a.x_t = p.x_t; a.x_b = p.x_b; a.z_t = p.z_t; a.z_b = p.z_b; a.d_t = p.delta_t; a.d_b = p.delta_b;
  a.bm_t = p.Bm_t; a.bm_b = p.Bm_b; a.cm_t = p.Cm_t; a.cm_b = p.Cm_b;
  a.A = p.A; a.D = p.D; a.dt_bias = p.dt_bias; a.conv_w = p.conv_w; a.conv_b = p.conv_b;
  a.done = p.done; a.first = p.first; a.h0 = p.h0; a.win0 = p.win0;
  return a;
}

int block_threads(const Args& a, bool grad) { return ssm_block_threads(a.per, a.Q, grad); }
static_assert(ssm_bwd_lds(kMaxStates / 4, 64) <= 64 * 1024, "one wavefront of the most states");

int set_chunks(Args& a, bool grad) {
  const long waves = a.B * a.G * ((a.per + 63) / 64);
  a.chunk = (int)ssm_chunk(a.T, a.B, a.G, a.per, a.N, grad);
  a.chunks = (a.T + a.chunk - 1) / a.chunk;
  PH_REQUIRE(a.chunks * waves < (1L << 31), "ssm: %ld sequences of %ld channels in %ld chunks of time", a.B, a.C, a.chunks);
  return PH_OK;
}

template <typename T>
int fwd_t(Args& a, hipStream_t st) {
  const int nt = block_threads(a, false);
  const size_t lds = ssm_fwd_lds(a.Q, nt);
  a.blocks_c = (unsigned)((a.per + nt - 1) / nt);
  const dim3 blocks = grid_rows((unsigned)(a.chunks * a.B * a.G * a.blocks_c));
  const int most = (kSteps * 8 * a.Q + nt - 1) / nt;
  if (a.chunks > 1) {
    if (most <= 1) k_ssm_fwd<T, true, 1><<<blocks, nt, lds, st>>>(a);
    else if (most <= 4) k_ssm_fwd<T, true, 4><<<blocks, nt, lds, st>>>(a);
    else k_ssm_fwd<T, true, 16><<<blocks, nt, lds, st>>>(a);
    PH_LAUNCH_CHECK();
    k_ssm_join<<<ceil_div((size_t)(a.B * a.C * 4 * a.Q), 256), 256, 0, st>>>(a);
    PH_LAUNCH_CHECK();
  }
  if (most <= 1) k_ssm_fwd<T, false, 1><<<blocks, nt, lds, st>>>(a);
  else if (most <= 4) k_ssm_fwd<T, false, 4><<<blocks, nt, lds, st>>>(a);
  else k_ssm_fwd<T, false, 16><<<blocks, nt, lds, st>>>(a);
  PH_LAUNCH_CHECK();
  if (a.win_out && !a.win_here) {
    k_ssm_window<T><<<ceil_div((size_t)(a.B * a.C), 256), 256, 0, st>>>(a);
    PH_LAUNCH_CHECK();
  }
  return PH_OK;
}

template <typename T>
int bwd_t(Args& a, GradArgs& ga, int nt, const ParOut& po, hipStream_t st) {
  const int most = (kSteps * 8 * a.Q + nt - 1) / nt;
  if (a.chunks > 1) {
    const unsigned blocks = (unsigned)(a.chunks * a.B * a.G * a.blocks_c);
    if (most <= 1) k_ssm_bwd_local<T, 1><<<blocks, nt, ssm_fwd_lds(a.Q, nt), st>>>(a, ga);
    else if (most <= 4) k_ssm_bwd_local<T, 4><<<blocks, nt, ssm_fwd_lds(a.Q, nt), st>>>(a, ga);
    else k_ssm_bwd_local<T, 16><<<blocks, nt, ssm_fwd_lds(a.Q, nt), st>>>(a, ga);
    PH_LAUNCH_CHECK();
    k_ssm_bwd_join<<<ceil_div((size_t)(a.B * a.C * 4 * a.Q), 256), 256, 0, st>>>(a, ga);
    PH_LAUNCH_CHECK();
  }
  const unsigned blocks = (unsigned)(ga.rows * a.G * a.blocks_c);
  if (most <= 1) k_ssm_bwd<T, 1><<<blocks, nt, ssm_bwd_lds(a.Q, nt), st>>>(a, ga);
  else if (most <= 4) k_ssm_bwd<T, 4><<<blocks, nt, ssm_bwd_lds(a.Q, nt), st>>>(a, ga);
  else k_ssm_bwd<T, 16><<<blocks, nt, ssm_bwd_lds(a.Q, nt), st>>>(a, ga);
  PH_LAUNCH_CHECK();
  if (a.chunks > 1 && a.K > 1 && ga.dx) {
    k_ssm_halo<T><<<ceil_div((size_t)((a.chunks - 1) * a.B * (a.K - 1) * a.C), 256), 256, 0, st>>>(a, ga);
    PH_LAUNCH_CHECK();
  }
  if (ga.bc) {
    const unsigned blocks = ceil_div((size_t)a.T * a.B * a.G * 2 * a.N, 256);
    k_ssm_fold_bc<T><<<blocks < 8192 ? blocks : 8192, 256, 0, st>>>(a, ga);
    PH_LAUNCH_CHECK();
  }
  const long CP = a.C * ga.P;
  const size_t folds = (size_t)(CP + 63) / 64, most_folds = 1u << 20;  // (2^32 threads or more would not all start)
  k_ssm_fold_par<<<(unsigned)(folds < most_folds ? folds : most_folds), 256, 0, st>>>(ga.par, ga.rows, CP, a.N, a.K, ga.P, po);
  PH_LAUNCH_CHECK();
  return PH_OK;
}

template <typename T>
int step_t(const Args& a, float* h, float* win, hipStream_t st) {
  const long w = (a.C + 63) / 64;
  const int nt = 64 * (int)(w < 4 ? w : 4);
  const long nblk = (a.C + nt - 1) / nt;
  // sequences of a block: what it loads once (decays, taps) is worth a few, as long as eight blocks are left for a CU
  long per_block = a.B * nblk / 2048;
  per_block = per_block < 1 ? 1 : per_block > 8 ? 8 : per_block;
  const long blocks = nblk * ((a.B + per_block - 1) / per_block);
  PH_REQUIRE(blocks < (1L << 31), "ssm_step: %ld sequences of %ld channels", a.B, a.C);
  const size_t lds = (size_t)(2 + a.Q) * nt * 4;
  const size_t ea = 4 * sizeof(T);  // a quad of B or C
  const bool vec = a.N % 4 == 0 && ((uintptr_t)h % 16) == 0 && ((uintptr_t)a.A % 16) == 0 && ((uintptr_t)a.Bm % ea) == 0 &&
                   ((uintptr_t)a.Cm % ea) == 0 && a.bm_b % 4 == 0 && a.cm_b % 4 == 0;
  const int qt = vec && (a.Q == 1 || a.Q == 2 || a.Q == 4) ? a.Q : 0;
  if (qt == 1) k_ssm_step<T, 1><<<(unsigned)blocks, nt, lds, st>>>(a, h, win, (int)per_block);
  else if (qt == 2) k_ssm_step<T, 2><<<(unsigned)blocks, nt, lds, st>>>(a, h, win, (int)per_block);
  else if (qt == 4) k_ssm_step<T, 4><<<(unsigned)blocks, nt, lds, st>>>(a, h, win, (int)per_block);
  else k_ssm_step<T, 0><<<(unsigned)blocks, nt, lds, st>>>(a, h, win, (int)per_block);
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
  return (p->T + kSteps - 1) / kSteps * p->B * p->C * ((p->N + 3) / 4 * 4);
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
  PH_TRY(set_chunks(a, false));
  a.win_out = a.K > 1 ? win_out : nullptr;
  // with several chunks the first one may still read the window that the last would overwrite
  a.win_here = a.win_out && (a.chunks == 1 || a.win_out != a.win0);
  if (a.chunks > 1) {
    const size_t nh = (size_t)a.chunks * a.B * a.C * 4 * a.Q, nd = (size_t)a.chunks * a.B * a.C;
    float* ws = (float*)scratch(kSlotSsm, (nh + nd) * 4);
    if (!ws) return PH_ERR_NOMEM;
    a.hloc = ws;
    a.dsum = ws + nh;
  }
  return p->dtype == PH_BF16 ? fwd_t<uint16_t>(a, st) : fwd_t<float>(a, st);
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
  PH_TRY(set_chunks(a, true));
  GradArgs ga{};
  ga.dy = dy; ga.dy_t = dy_t; ga.dy_b = dy_b; ga.keep = keep;
  ga.dx = g->dx; ga.dx_t = g->dx_t; ga.dx_b = g->dx_b;
  ga.dz = p->z ? g->dz : nullptr; ga.dz_t = g->dz_t; ga.dz_b = g->dz_b;
  ga.ddelta = g->ddelta; ga.dd_t = g->ddelta_t; ga.dd_b = g->ddelta_b;
  ga.dB = g->dBm; ga.db_t = g->dBm_t; ga.db_b = g->dBm_b;
  ga.dC = g->dCm; ga.dc_t = g->dCm_t; ga.dc_b = g->dCm_b;
  ga.P = (int)(a.N + a.K + 3);
  const int nt = block_threads(a, true);
  const long G = a.G, bc = (a.per + nt - 1) / nt;
  a.blocks_c = (unsigned)bc;
  // blocks of a channel block: as many as run at a time, with as equal shares of the items as there are
  const long items = a.B * a.chunks, most = ssm_resident(nt) / (G * bc) > 0 ? ssm_resident(nt) / (G * bc) : 1;
  const long rounds = (items + most - 1) / most;
  ga.rows = (items + rounds - 1) / rounds;
  if (ga.rows < 1) ga.rows = 1;
  const size_t nh = a.chunks > 1 ? (size_t)a.chunks * a.B * a.C * 4 * a.Q : 0, nd = a.chunks > 1 ? (size_t)a.chunks * a.B * a.C : 0;
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
  return p->dtype == PH_BF16 ? bwd_t<uint16_t>(a, ga, nt, po, st) : bwd_t<float>(a, ga, nt, po, st);
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
  hipStream_t st = as_stream(stream);
  return p->dtype == PH_BF16 ? step_t<uint16_t>(a, h, win, st) : step_t<float>(a, h, win, st);
}
