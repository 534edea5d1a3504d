// Draw of one entry per row of logits after temperature, top-k, top-p and min-p, from a given number u.
//
// What the filters leave is every entry above a threshold key, and of those at the threshold the ones up to an index:
// top-k's threshold is the k-th largest key, top-p's the one at which the mass of the larger ones reaches p of the total.
// Neither needs the row sorted: a key is a 32-bit number that orders like the logit; the keys among which the threshold lies are
// narrowed down by how much (count, or mass) is above some, until few enough are left to be compared with each other. What is
// left of the row is then summed up in the order of its indices to where the sum exceeds u times the total.
//
// Masses are exp((l - max) / temperature) from 64-bit floating point, held as whole numbers of 2^-bits with as many bits as the
// sum of A of them has room for (45 at 131072 entries, 51 up to 2048): sums do not depend on their order, so the
// borders that u and p are compared with are the same however the row is split.
//
// Bound by vector instructions. Measured, with the calls' own 12 us: 4096 rows of 1000 fp32 logits 31 us with filters mixed, 16.8
// without any, 23.6 with top-k, 31.7 with top-p: of some 2340 vector instructions a row a quarter are the 64-bit exponentials and their
// units (some 40 an entry), the others narrow the keys down and compare what is left. 64 rows of 32768 bf16, a block each, 29,
// 26 and 64 us; of 131072 over sixteen blocks each 40, 46 and 100, mixed 106, half of it the last launch, where all wavefronts of 64 blocks
// compare what is listed. 48 rows of 18 in the time of the launch.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "routes.hpp"
#include "spans.hpp"

namespace ph {
namespace {

typedef unsigned long long u64;

__device__ __forceinline__ float ldf(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float ldf(const float* p) { return *p; }

// Orders like the logit, both zeros alike; 0 for what is never taken.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (!(v > -INFINITY)) return 0;  // -inf, NaN
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __builtin_bit_cast(float, k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// A row's parameters, with the filters that are off in a form that lets everything pass.
struct Par {
  double c, p;  // log2(e) / temperature
  float minp, u;
  long k;
  bool greedy;
};
struct DrawArgs {
  const void* x;
  long ld, N;
  int A, bits;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  int* act;
  float* logp;
};
__device__ __forceinline__ Par par_of(const DrawArgs& a, long n) {
  Par r;
  const float t = a.temperature ? a.temperature[n] : 1.f, p = a.top_p ? a.top_p[n] : 1.f, m = a.min_p ? a.min_p[n] : 0.f;
  r.c = 1.4426950408889634074 / (t > 0.f ? (double)t : 1.0);
  r.k = a.top_k && a.top_k[n] > 0 ? a.top_k[n] : a.A;
  r.greedy = t == 0.f || p <= 0.f;
  r.p = p < 1.f ? (double)p : 1.0;
  r.minp = m > 0.f ? (m < 1.f ? m : 1.f) : 0.f;
  r.u = a.u[n];
  return r;
}
// 2^y for y <= 0 as a factor in 0.7..1.42 and an exponent: exp by its series, to z^12 for |z| <= ln 2 / 2 (what is left out is
// below 2^-52).
struct Mass {
  double r;
  int n;
};
__device__ __forceinline__ Mass mass_of(uint32_t key, uint32_t top, double c) {  // c = log2(e) / temperature
  const double d = (double)logit_of(key) - (double)logit_of(top);
  double y = d * c;
  y = y > -1000.0 ? y : -1000.0;
  const double n = rint(y), z = (y - n) * 0.6931471805599453094;
  double p = 1.0 / 479001600;
  p = fma(p, z, 1.0 / 39916800);
  p = fma(p, z, 1.0 / 3628800);
  p = fma(p, z, 1.0 / 362880);
  p = fma(p, z, 1.0 / 40320);
  p = fma(p, z, 1.0 / 5040);
  p = fma(p, z, 1.0 / 720);
  p = fma(p, z, 1.0 / 120);
  p = fma(p, z, 1.0 / 24);
  p = fma(p, z, 1.0 / 6);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  Mass m = {p, (int)n};
  if (key == top) m = {1.0, 0};  // of an infinite logit too, whose difference is none
  return m;
}
// The same by a table of 2^(i / 1024), i = 0..1023: the series ends with z^3 for |z| <= ln 2 / 2048 (left out: below 2^-50), half the
// instructions. For rows that are worth the table.
constexpr int kTable = 1024;
__device__ __forceinline__ Mass mass_of(uint32_t key, uint32_t top, double c, const double* table) {
  double y = ((double)logit_of(key) - (double)logit_of(top)) * (c * kTable);
  y = y > -1000.0 * kTable ? y : -1000.0 * kTable;
  const double n = rint(y), z = (y - n) * (0.6931471805599453094 / kTable);
  const int i = (int)n;
  Mass m = {table[i & (kTable - 1)] * fma(z, fma(z, fma(z, 1.0 / 6, 0.5), 1.0), 1.0), i >> 10};
  if (key == top) m = {1.0, 0};
  return m;
}
// In units of 2^-bits, to the nearest.
__device__ __forceinline__ u64 units(Mass m, int bits) {
  const u64 b = __builtin_bit_cast(u64, m.r);
  const int shift = 52 - ((int)(b >> 52) - 1023) - m.n - bits;  // the double's sign is 0
  const u64 f = (b & 0xfffffffffffffull) | 0x10000000000000ull;
  return shift > 53 ? 0 : (f + (1ull << (shift - 1))) >> shift;
}
// The logarithm of an entry's share of the total: from its logit, not from its units, of which it may have few.
__device__ __forceinline__ float log_share(uint32_t key, uint32_t top, double c, u64 total, int bits) {
  const double d = key == top ? 0.0 : ((double)logit_of(key) - (double)logit_of(top)) * c * 0.6931471805599453094;
  return (float)(d - log(ldexp((double)total, -bits)));
}
// What an entry has to have by min_p, in these units.
__device__ __forceinline__ u64 least(float minp, int bits) { return (u64)ceil(ldexp((double)minp, bits)); }

// ---- sums over a wavefront --------------------------------------------------------------------------------
template <int CTL> __device__ __forceinline__ u64 dpp64(u64 v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTL, 0xF, 0xF, true);
  return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
  v += dpp64<0xB1>(v);
  v += dpp64<0x4E>(v);
  v += dpp64<0x141>(v);
  v += dpp64<0x140>(v);
  float a = __builtin_bit_cast(float, (uint32_t)v), b = __builtin_bit_cast(float, (uint32_t)(v >> 32)), a2 = a, b2 = b;
  swap16(a, a2, b, b2);
  auto join = [](float lo, float hi) { return ((u64)__builtin_bit_cast(uint32_t, hi) << 32) | __builtin_bit_cast(uint32_t, lo); };
  v = join(a, b) + join(a2, b2);
  a = __builtin_bit_cast(float, (uint32_t)v);
  b = __builtin_bit_cast(float, (uint32_t)(v >> 32));
  a2 = a;
  b2 = b;
  swap32(a, a2, b, b2);
  return join(a, b) + join(a2, b2);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v) {  // inclusive
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 o = __shfl_up(v, d);
    if (l >= d) v += o;
  }
  return v;
}

// Order of two entries: the larger key, of equal ones the lower index.
__device__ __forceinline__ u64 order_of(uint32_t key, uint32_t index) { return (u64)key << 32 | (0xffffffffu - index); }

// ---- rows in the registers of a wavefront ---------------------------------------------------------------------
// Entry 64 e + lane in register e.
struct WaveLds {
  u64 order[64], mass[64];
};
template <typename T, int E> __global__ void __launch_bounds__(256, 4) k_draw_wave(const DrawArgs a) {
  __shared__ WaveLds lds[4];
  int l = threadIdx.x & 63;
  // what goes by the lane's number is formed again from here on, and does not wait in registers
  auto renew = [&] { asm volatile("" : "+v"(l)); };
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  WaveLds& L = lds[w];
  for (long n = (long)blockIdx.x * 4 + w; n < a.N; n += (long)gridDim.x * 4) {
    const T* row = (const T*)a.x + n * a.ld;
    uint32_t key[E], top = 0;
    {
      T x[E];
#pragma unroll
      for (int e = 0; e < E; e++) x[e] = row[64 * e + l < a.A ? 64 * e + l : 0];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const uint32_t k = key_of(ldf(&x[e]));
        key[e] = 64 * e + l < a.A ? k : 0;
        top = key[e] > top ? key[e] : top;
      }
    }
    renew();
    const Par par = par_of(a, n);
    top = (uint32_t)__builtin_amdgcn_readfirstlane((int)wave_max(top));
    int act = -1;
    float logp = -INFINITY;
    // the entries at `key` in the order of their indices: the index of the count-th (from 1). Few rows ask, so it reads them again.
    auto index_at = [&](uint32_t k, long count) {
      int cut = a.A;
#pragma unroll 1
      for (int at = 0; at < a.A && count > 0; at += 64) {
        const u64 on = __ballot(at + l < a.A && key_of(ldf(row + (at + l < a.A ? at + l : 0))) == k);
        const int c = __popcll(on);
        if (count <= c) {
          const u64 is = __ballot(((on >> l) & 1) && __popcll(on & ((2ull << l) - 1)) == count);
          cut = at + __ffsll((unsigned long long)is) - 1;
        }
        count -= c;
      }
      return cut;
    };
    if (top == 0) {
    } else if (par.greedy) {
      act = index_at(top, 1);
      logp = 0.f;
    } else {
      uint32_t thr = 1;
      int cut = a.A;
      auto left = [&](int e) { return (key[e] > thr) | ((key[e] == thr) & (64 * e + l <= cut)); };
      if (E > 1 && par.k < a.A) {
        // at least k keys are lo and above, fewer hi and above: until there are k, or equal ones at the border
        auto count = [&](uint32_t c) {
          int n = 0;
#pragma unroll
          for (int e = 0; e < E; e++) n += __popcll(__ballot(key[e] >= c));
          return n;
        };
        uint32_t lo = 1, hi = top;
        int at_least = count(1), above = 0;
        if (at_least > par.k) {
          above = count(top);
          if (above >= par.k) {  // the largest alone are as many
            lo = top;
            at_least = above;
            above = 0;
          } else {
            while (at_least > par.k && hi - lo > 1) {
              const uint32_t mid = lo + (hi - lo) / 2;
              const int c = count(mid);
              if (c >= par.k) {
                lo = mid;
                at_least = c;
              } else {
                hi = mid;
                above = c;
              }
            }
          }
          thr = lo;
          if (at_least > par.k) cut = index_at(thr, par.k - above);
        }
      }
      renew();
      u64 m[E], total = 0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const u64 x = units(mass_of(key[e], top, par.c), a.bits);
        m[e] = (key[e] != 0) & left(e) ? x : 0;
        total += m[e];
        if (E > 4 && e % 2) __builtin_amdgcn_sched_barrier(0);  // or all registers' series run side by side, and do not fit
      }
      renew();
      // of at most 64 entries in LDS, lane i's: how many and how much mass is in front of it
      auto compare = [&](int count, u64 mine, int& rank, u64& before) {
        for (int j = 0; j < count; j++) {
          const bool first = L.order[j] > mine;
          rank += first;
          before += first ? L.mass[j] : 0;
        }
      };
      if constexpr (E == 1) {
        if (par.k < a.A || par.p < 1.0) {
          const u64 mine = order_of(key[0], l);
          L.order[l] = mine;
          L.mass[l] = m[0];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          int rank = 0;
          u64 before = 0;
          compare(a.A, mine, rank, before);
          if (rank >= par.k) m[0] = 0;
          if (par.p < 1.0) {
            const u64 want = (u64)ceil(par.p * (double)wave_sum(m[0]));
            if (before >= want) m[0] = 0;
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
      } else if (par.p < 1.0) {
        total = wave_sum(total);
        const u64 want = (u64)ceil(par.p * (double)total);
        // the threshold lies in lo + 1..hi: at least `want` is above lo, less above hi
        uint32_t lo = thr - 1, hi = top;
        long over_lo = (long)a.A, over_hi = 0;  // entries above them
        u64 above_hi = 0;
        while (over_lo - over_hi > 64 && hi - lo > 1) {
          const uint32_t mid = lo + (hi - lo) / 2;
          u64 sum = 0;
          long cnt = 0;
#pragma unroll
          for (int e = 0; e < E; e++) {
            const bool on = key[e] > mid;
            sum += on ? m[e] : 0;
            cnt += __popcll(__ballot(on));
          }
          sum = wave_sum(sum);
          if (sum >= want) {
            lo = mid;
            over_lo = cnt;
          } else {
            hi = mid;
            over_hi = cnt;
            above_hi = sum;
          }
        }
        renew();
        int count = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
          const bool on = key[e] > lo && key[e] <= hi && m[e];
          const u64 all = __ballot(on);
          const int at = count + __popcll(all & ((1ull << l) - 1));
          if (on && at < 64) {
            L.order[at] = order_of(key[e], 64 * e + l);
            L.mass[at] = m[e];
          }
          count += __popcll(all);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (count <= 64) {
          const u64 mine = l < count ? L.order[l] : 0;
          int rank = 0;
          u64 before = above_hi;
          compare(count, mine, rank, before);
          const u64 kept = __ballot(l < count && before < want);
          const int last = __ffsll((unsigned long long)__ballot(l < count && rank == __popcll(kept) - 1)) - 1;
          const u64 o = __shfl(mine, last);
          thr = (uint32_t)(o >> 32);
          cut = (int)(0xffffffffu - (uint32_t)o);
        } else {  // equal ones, of which the first few are left (top-k may have cut them already)
          const u64 each = units(mass_of(hi, top, par.c), a.bits), of = (want - above_hi + each - 1) / each;
          const int at = index_at(hi, (long)of);
          if (hi > thr) cut = a.A;
          thr = hi;
          cut = at < cut ? at : cut;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
      renew();
      const u64 need = least(par.minp, a.bits);
      // in the order of the indices: through[e] is the lane's share of the first e + 1 registers
      u64 through[E], run = 0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        m[e] = left(e) & (m[e] >= need) ? m[e] : 0;
        run += m[e];
        through[e] = run;
      }
      total = wave_sum(run);
      const u64 target = (u64)((double)par.u * (double)total);  // a sum exceeds u total where it exceeds this
      int tile = 0;  // registers that end at or below the target
      run = 0;
#pragma unroll
      for (int step = E / 2; step > 0; step /= 2) {
        u64 x = 0;
#pragma unroll
        for (int e = 0; e < E; e++) x = e == tile + step - 1 ? through[e] : x;
        x = wave_sum(x);
        if (x <= target && x < total) {
          tile += step;
          run = x;
        }
      }
      u64 mine = 0;
#pragma unroll
      for (int e = 0; e < E; e++) mine = e == tile ? m[e] : mine;
      tile = __builtin_amdgcn_readfirstlane(tile);
      const float logit = ldf(row + (64 * tile + l < a.A ? 64 * tile + l : 0));  // again: the keys did not wait in registers
      const u64 at = run + wave_scan(mine);
      u64 hit = __ballot(mine > 0 && at > target);
      if (!hit) hit = 1ull << (63 - __clzll((long long)__ballot(mine > 0)));  // u rounded up to 1: the last
      const int lane = __ffsll((unsigned long long)hit) - 1;
      act = 64 * tile + lane;
      logp = log_share(key_of(__shfl(logit, lane)), top, par.c, total, a.bits);
    }
    if (l == 0) {
      a.act[n] = act;
      if (a.logp) a.logp[n] = logp;
    }
  }
}

// ---- wide rows: a block each ----------------------------------------------------------------------------------
// The wavefronts take a part of the row each, lanes 16 bytes at a time.
constexpr int kWide = 1024, kBins = 2048, kList = 1024;

struct WideLds {
  u64 bins[kBins], wave[16], above;
  u64 order[kList], mass[kList];
  uint32_t key;
  int found, count;
};

// The largest bin b with sum(bins[b..]) >= want, in every thread: found, and above = sum(bins[b + 1 ..]). Every thread calls.
__device__ __forceinline__ void pick_bin(WideLds& L, int nbins, u64 want, int& bin, u64& above) {
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  __syncthreads();
  if (tid == 0) L.found = 0, L.above = 0;
  // thread t has the bins nbins - 1 - 2 t and the one below
  const int b0 = nbins - 1 - 2 * tid;
  const u64 x0 = b0 >= 0 ? L.bins[b0] : 0, x1 = b0 >= 1 ? L.bins[b0 - 1] : 0;
  const u64 incl = wave_scan(x0 + x1);
  if (l == 63) L.wave[w] = incl;
  __syncthreads();
  u64 before = incl - x0 - x1;
  for (int i = 0; i < w; i++) before += L.wave[i];
  if (before < want) {
    if (before + x0 >= want) {
      L.found = b0;
      L.above = before;
    } else if (before + x0 + x1 >= want) {
      L.found = b0 - 1;
      L.above = before + x0;
    }
  }
  __syncthreads();
  bin = L.found;
  above = L.above;
}

template <typename T> struct Row {
  static constexpr int V = 16 / sizeof(T);
  const T* x;
  int from, to;  // this wavefront's entries
  __device__ __forceinline__ Row(const DrawArgs& a, long n, int w, int parts) {
    x = (const T*)a.x + n * a.ld;
    const int part = size(a.A, parts);
    from = w * part < a.A ? w * part : a.A;
    to = from + part < a.A ? from + part : a.A;
  }
  static __device__ __forceinline__ int size(int A, int parts) { return (A + parts * 64 * V - 1) / (parts * 64 * V) * (64 * V); }
  // The keys of the lane's entries at `at` + V lane .., 0 behind the part's end.
  __device__ __forceinline__ void keys(int at, uint32_t* k) const {
    const int i = at + V * (threadIdx.x & 63);
    T v[V];
    if (i + V <= to) {
      __builtin_memcpy(v, x + i, 16);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) v[j] = i + j < to ? x[i + j] : T(0);
    }
#pragma unroll
    for (int j = 0; j < V; j++) k[j] = i + j < to ? key_of(raw(v[j])) : 0;
  }
  static __device__ __forceinline__ float raw(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ float raw(float v) { return v; }
  // f(key, index) for every entry of the lane that may be taken; whole wavefronts, so that f may exchange values.
  template <typename F> __device__ __forceinline__ void each(F f) const {
    for (int at = from; at < to; at += 64 * V) {
      uint32_t k[V];
      keys(at, k);
#pragma unroll
      for (int j = 0; j < V; j++) f(k[j], at + V * (int)(threadIdx.x & 63) + j);
    }
  }
};

// Bins of equal width in the logit below the largest, down to masses of 2^-bits; they fall with the key.
struct Bins {
  float ltop, per;
  uint32_t top;
  __device__ __forceinline__ Bins(const DrawArgs& a, const Par& par, uint32_t t) : top(t) {
    ltop = logit_of(t);
    per = (float)(kBins - 1) / (float)(((double)a.bits + 1) / par.c);
  }
  __device__ __forceinline__ int operator()(uint32_t k) const {
    const float d = (ltop - logit_of(k)) * per;
    return k == top || !(d > 0.f) ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;
  }
};

__device__ __forceinline__ u64 block_sum(WideLds& L, u64 v) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  v = wave_sum(v);
  __syncthreads();
  if (l == 0) L.wave[w] = v;
  __syncthreads();
  u64 all = 0;
  for (int i = 0; i < 16; i++) all += L.wave[i];
  return all;
}

// The thread's entry of the list: how many and how much mass is in front of it.
__device__ __forceinline__ void compare(const WideLds& L, u64 mine, int& rank, u64& before) {
  const int count = L.count;
  for (int j = 0; j < count; j++) {
    const bool first = L.order[j] > mine;
    rank += first;
    before += first ? L.mass[j] : 0;
  }
}
// The entry that `is_it` holds for is the last that is left.
__device__ __forceinline__ void cut_at(WideLds& L, bool is_it, u64 mine, uint32_t& thr, int& cut) {
  if (is_it) {
    L.key = (uint32_t)(mine >> 32);
    L.found = (int)(0xffffffffu - (uint32_t)mine);
  }
  __syncthreads();
  thr = L.key;
  cut = L.found;
}

// All that top-k leaves is in the list, one entry a thread: the rest of the filters and the draw.
__device__ __forceinline__ void draw_listed(WideLds& L, const DrawArgs& a, long n, const Par& par, uint32_t top, uint32_t thr, int cut) {
  const int tid = threadIdx.x, count = L.count;
  const u64 mine = tid < count ? L.order[tid] : 0;
  const uint32_t k = (uint32_t)(mine >> 32);
  const int i = (int)(0xffffffffu - (uint32_t)mine);
  u64 m = tid < count && (k > thr || (k == thr && i <= cut)) ? L.mass[tid] : 0;
  const u64 of = block_sum(L, m);
  if (par.p < 1.0) {
    int rank = 0;
    u64 before = 0;
    compare(L, mine, rank, before);
    if (before >= (u64)ceil(par.p * (double)of)) m = 0;
  }
  if (m < least(par.minp, a.bits)) m = 0;
  const u64 total = block_sum(L, m);
  L.mass[tid] = m;
  if (tid == 0) L.found = a.A;
  __syncthreads();
  const u64 target = (u64)((double)par.u * (double)total);
  u64 run = 0;  // up to this entry, in the order of the indices
  for (int j = 0; j < count; j++) run += (uint32_t)L.order[j] >= (uint32_t)mine ? L.mass[j] : 0;
  if (m && (run > target || run == total)) atomicMin(&L.found, i);
  __syncthreads();
  if (m && i == L.found) {
    a.act[n] = i;
    if (a.logp) a.logp[n] = log_share(k, top, par.c, total, a.bits);
  }
}

// The wavefront's part of the row is where the sum, `before` in front of it, exceeds the target.
template <typename T, typename F>
__device__ __forceinline__ void draw_in_part(const DrawArgs& a, long n, const Row<T>& row, F left_at, u64 before, u64 target, u64 total,
                                             uint32_t top, double c) {
  constexpr int V = Row<T>::V;
  const int l = threadIdx.x & 63;
  for (int at = row.from; at < row.to; at += 64 * V) {
    uint32_t k[V];
    u64 m[V], here = 0;
    row.keys(at, k);
#pragma unroll
    for (int j = 0; j < V; j++) here += m[j] = left_at(k[j], at + V * l + j);
    const u64 incl = wave_scan(here), all = __shfl(incl, 63);
    if (all && (before + all > target || before + all == total)) {
      u64 run = before + incl - here;
      int first = -1;  // of the lane's entries: the first that exceeds, or (u rounded up to 1) the last there is
      uint32_t got = 0;
#pragma unroll
      for (int j = 0; j < V; j++) {
        run += m[j];
        if (m[j] && (run > target || run == total) && first < 0) {
          first = j;
          got = k[j];
        }
      }
      const u64 who = __ballot(first >= 0);
      if (l == __ffsll((unsigned long long)who) - 1) {
        a.act[n] = at + V * l + first;
        if (a.logp) a.logp[n] = log_share(got, top, c, total, a.bits);
      }
      break;
    }
    before += all;
  }
}

template <typename T> __device__ __forceinline__ void draw_row(WideLds& L, const double* table, const DrawArgs& a, long n) {
  constexpr int V = Row<T>::V;
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Row<T> row(a, n, w, 16);
  const Par par = par_of(a, n);
  __syncthreads();
  uint32_t best = 0;  // of the thread
  int valid = 0;
  row.each([&](uint32_t k, int) {
    best = k > best ? k : best;
    valid += k != 0;
  });
  uint32_t top = wave_max(best);
  if (l == 0) L.wave[w] = top;
  __syncthreads();
  for (int i = 0; i < 16; i++) top = (uint32_t)L.wave[i] > top ? (uint32_t)L.wave[i] : top;
  if (top == 0) {
    if (tid == 0) {
      a.act[n] = -1;
      if (a.logp) a.logp[n] = -INFINITY;
    }
    return;
  }
  // the index of the count-th entry (from 1) with this key, by the wavefronts' parts
  auto index_at = [&](uint32_t k, u64 count) {
    int c = 0;
    row.each([&](uint32_t x, int) { c += x == k; });
    const u64 mine = wave_sum((u64)c);
    __syncthreads();
    if (l == 0) L.wave[w] = mine;
    if (tid == 0) L.found = a.A;
    __syncthreads();
    u64 before = 0;
    for (int i = 0; i < w; i++) before += L.wave[i];
    if (before < count && count <= before + mine) {
      for (int at = row.from; at < row.to; at += 64 * V) {
        uint32_t x[V];
        row.keys(at, x);
        int here = 0;
#pragma unroll
        for (int j = 0; j < V; j++) here += x[j] == k;
        const u64 incl = wave_scan((u64)here);
        u64 rank = before + incl - here;
#pragma unroll
        for (int j = 0; j < V; j++)
          if (x[j] == k && ++rank == count) L.found = at + V * l + j;
        before += __shfl(incl, 63);
      }
    }
    __syncthreads();
    return L.found;
  };
  if (par.greedy) {
    const int i = index_at(top, 1);
    if (tid == 0) {
      a.act[n] = i;
      if (a.logp) a.logp[n] = 0.f;
    }
    return;
  }
  uint32_t thr = 1;
  int cut = a.A;
  auto left = [&](uint32_t k, int i) { return k > thr || (k == thr && i <= cut); };
  auto mass_at = [&](uint32_t k) { return units(mass_of(k, top, par.c, table), a.bits); };
  const u64 need = least(par.minp, a.bits);
  // The entries between two keys into the list, in any order; false (and no list) if there are too many.
  auto gather = [&](uint32_t lo, uint32_t hi, bool mass) {  // lo <= key <= hi
    __syncthreads();
    if (tid == 0) L.count = 0;
    __syncthreads();
    row.each([&](uint32_t k, int i) {
      if (k && k >= lo && k <= hi && left(k, i)) {
        const int at = atomicAdd(&L.count, 1);
        if (at < kList) {
          L.order[at] = order_of(k, (uint32_t)i);
          if (mass) L.mass[at] = mass_at(k);
        }
      }
    });
    __syncthreads();
    return L.count <= kList;
  };
  // The threshold by digits of the key of 11, 11 and 10 bits, a histogram in LDS each: the largest key at and above which there is
  // `want` (entries, or mass), and what is wanted of those at it.
  auto select = [&](bool mass, u64 want, u64& rest) {
    uint32_t key = 0;
    int have = 0;  // bits of the key that are known
    for (int d = 0; d < 3; d++) {
      const int bits = d < 2 ? 11 : 10, shift = 32 - have - bits;
      __syncthreads();
      for (int i = tid; i < kBins; i += kWide) L.bins[i] = 0;
      __syncthreads();
      row.each([&](uint32_t k, int i) {
        if (!k || !left(k, i) || (have && (k >> (32 - have)) != key >> (32 - have))) return;
        atomicAdd(&L.bins[k >> shift & ((1u << bits) - 1)], mass ? mass_at(k) : 1ull);
      });
      int bin;
      u64 above;
      pick_bin(L, 1 << bits, want, bin, above);
      want -= above;
      key |= (uint32_t)bin << shift;
      have += bits;
    }
    rest = want;
    return key;
  };
  bool listed = false;  // all that is left is in the list
  if (par.k < a.A && block_sum(L, (u64)valid) > (u64)par.k) {
    if (par.k <= kWide) {
      // the k-th largest of the threads' largest keys bounds the k-th largest of all from below
      uint32_t cur = 0;
      for (int bit = 31; bit >= (sizeof(T) == 2 ? 16 : 0); bit--)
        if (__syncthreads_count(best >= (cur | (1u << bit))) >= par.k) cur |= 1u << bit;
      if (cur && gather(cur, top, true)) {
        const u64 mine = tid < L.count ? L.order[tid] : 0;
        int rank = 0;
        u64 before = 0;
        compare(L, mine, rank, before);
        cut_at(L, tid < L.count && rank == par.k - 1, mine, thr, cut);
        listed = true;
      }
    }
    if (!listed) {
      u64 rest;
      const uint32_t k = select(false, (u64)par.k, rest);
      cut = index_at(k, rest);
      thr = k;
    }
  }
  if (listed) {
    draw_listed(L, a, n, par, top, thr, cut);
    return;
  }
  if (par.p < 1.0) {
    // What falls into the bin where the threshold lies is few enough for the list, unless many are equal.
    const Bins bins(a, par, top);
    __syncthreads();
    for (int i = tid; i < kBins; i += kWide) L.bins[i] = 0;
    __syncthreads();
    u64 s = 0;
    row.each([&](uint32_t k, int i) {
      if (!k || !left(k, i)) return;
      const u64 m = mass_at(k);
      s += m;
      if (m) atomicAdd(&L.bins[kBins - 1 - bins(k)], m);
    });
    const u64 want = (u64)ceil(par.p * (double)block_sum(L, s));
    int bin;
    u64 above;
    pick_bin(L, kBins, want, bin, above);
    bin = kBins - 1 - bin;
    __syncthreads();
    if (tid == 0) L.count = 0;
    __syncthreads();
    row.each([&](uint32_t k, int i) {
      if (!k || bins(k) != bin || !left(k, i)) return;
      const int at = atomicAdd(&L.count, 1);
      if (at < kList) {
        L.order[at] = order_of(k, (uint32_t)i);
        L.mass[at] = mass_at(k);
      }
    });
    __syncthreads();
    if (L.count <= kList) {
      const u64 mine = tid < L.count ? L.order[tid] : 0;
      int rank = 0;
      u64 before = above;
      compare(L, mine, rank, before);
      const int kept = __syncthreads_count(tid < L.count && before < want);
      cut_at(L, tid < L.count && rank == kept - 1, mine, thr, cut);
    } else {
      u64 rest;
      const uint32_t k = select(true, want, rest);
      const u64 each = mass_at(k), of = each ? (rest + each - 1) / each : 1;
      const int at = index_at(k, of);
      if (k > thr) cut = a.A;
      thr = k;
      cut = at < cut ? at : cut;
    }
  }
  auto left_at = [&](uint32_t k, int i) {
    if (!k || !left(k, i)) return 0ull;
    const u64 m = mass_at(k);
    return m >= need ? m : 0ull;
  };
  u64 s = 0;
  row.each([&](uint32_t k, int i) { s += left_at(k, i); });
  const u64 mine = wave_sum(s);
  const u64 total = block_sum(L, s);  // L.wave: the wavefronts' sums
  u64 before = 0;
  for (int i = 0; i < w; i++) before += L.wave[i];
  const u64 target = (u64)((double)par.u * (double)total);
  if (mine && before <= target && (before + mine > target || before + mine == total))
    draw_in_part<T>(a, n, row, left_at, before, target, total, top, par.c);
}

template <typename T> __global__ void __launch_bounds__(kWide) k_draw_wide(const DrawArgs a) {
  __shared__ WideLds L;
  __shared__ double table[kTable];
  static_assert(kTable == kWide, "an entry each");
  table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
  for (long n = blockIdx.x; n < a.N; n += gridDim.x) draw_row<T>(L, table, a, n);
}

// ---- few wide rows: several blocks each -------------------------------------------------------------------------
// A row's entries in 64 parts, a wavefront each, 16 blocks to a row; what they find out goes through memory from one launch to the next:
//   k_split_keys   the largest key, how many may be taken, a lower bound of the k-th largest
//   k_split_masses top-k: the entries above that bound, listed; top-p: the masses by bins; neither: the parts' sums
//   k_split_bin    top-p: the bin where the threshold lies
//   k_split_border top-p: that bin's entries, listed, and the parts' sums of the ones above it
//   k_split_draw   the threshold among the listed, the draw; or all of it from the start, where a list is too short
// Whole numbers add up in any order, so the launches may use atomics.
constexpr int kSplit = 16, kParts = 64;
struct SplitRow {
  u64 bins[kBins], order[kList], mass[kList], sums[kParts], want, above;
  uint32_t top[kSplit], share[kSplit];
  int valid[kSplit], count, bin, greedy, pad;
};
enum SplitKind { kNone, kGreedy, kTopK, kTopP, kPlain, kFallBack };

struct SplitState {
  Par par;
  uint32_t top, bound;
  SplitKind kind;
  __device__ __forceinline__ SplitState(const DrawArgs& a, const SplitRow& r, long n) : par(par_of(a, n)), top(0), bound(0) {
    long valid = 0;
    bound = 0xffffffffu;
    for (int i = 0; i < kSplit; i++) {
      top = r.top[i] > top ? r.top[i] : top;
      bound = r.share[i] < bound ? r.share[i] : bound;
      valid += r.valid[i];
    }
    kind = top == 0 ? kNone : par.greedy ? kGreedy : par.k < valid ? (bound ? kTopK : kFallBack) : par.p < 1.0 ? kTopP : kPlain;
  }
};

template <typename T> __global__ void __launch_bounds__(256) k_split_keys(const DrawArgs a, SplitRow* rows) {
  __shared__ uint32_t tops[4];
  __shared__ int valids[4];
  const long n = blockIdx.y;
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x;
  SplitRow& r = rows[n];
  const Par par = par_of(a, n);
  for (int i = b * 256 + tid; i < kBins; i += kSplit * 256) r.bins[i] = 0;
  if (b == 0 && tid == 0) r.count = 0, r.greedy = a.A;
  const Row<T> row(a, n, 4 * b + w, kParts);
  uint32_t best = 0;
  int valid = 0;
  row.each([&](uint32_t k, int) {
    best = k > best ? k : best;
    valid += k != 0;
  });
  const uint32_t top = wave_max(best);
  const u64 v = wave_sum((u64)valid);
  if (l == 0) tops[w] = top, valids[w] = (int)v;
  // of the threads' largest keys the (k / blocks)-th: at least that many entries reach it, and in all at least k the least block's
  uint32_t share = 0;
  const int blocks = (a.A + 4 * Row<T>::size(a.A, kParts) - 1) / (4 * Row<T>::size(a.A, kParts));  // that have entries
  const long of = (par.k + blocks - 1) / blocks;
  if (!par.greedy && par.k <= kList && par.k < a.A) {
    for (int bit = 31; bit >= (sizeof(T) == 2 ? 16 : 0); bit--)
      if (__syncthreads_count(best >= (share | (1u << bit))) >= of) share |= 1u << bit;
  }
  if (b >= blocks) share = 0xffffffffu;
  __syncthreads();
  if (tid == 0) {
    uint32_t t = 0;
    int all = 0;
    for (int i = 0; i < 4; i++) {
      t = tops[i] > t ? tops[i] : t;
      all += valids[i];
    }
    r.top[b] = t;
    r.valid[b] = all;
    r.share[b] = share;
  }
}

// An entry into the row's list, while there is room.
__device__ __forceinline__ void list(SplitRow& r, uint32_t k, int i, u64 m) {
  const int at = atomicAdd(&r.count, 1);
  if (at < kList) {
    r.order[at] = order_of(k, (uint32_t)i);
    r.mass[at] = m;
  }
}

template <typename T> __global__ void __launch_bounds__(256) k_split_masses(const DrawArgs a, SplitRow* rows) {
  __shared__ double table[kTable];
  __shared__ u64 bins[kBins];
  const long n = blockIdx.y;
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x;
  SplitRow& r = rows[n];
  const SplitState s(a, r, n);
  if (s.kind == kNone || s.kind == kFallBack) return;
  const Row<T> row(a, n, 4 * b + w, kParts);
  if (s.kind == kGreedy) {
    int first = a.A;
    row.each([&](uint32_t k, int i) { first = k == s.top && i < first ? i : first; });
    if (first < a.A) atomicMin(&r.greedy, first);
    return;
  }
  for (int i = tid; i < kTable; i += 256) table[i] = exp2((double)i / kTable);
  for (int i = tid; i < kBins; i += 256) bins[i] = 0;
  __syncthreads();
  auto mass_at = [&](uint32_t k) { return units(mass_of(k, s.top, s.par.c, table), a.bits); };
  if (s.kind == kTopK) {
    row.each([&](uint32_t k, int i) {
      if (k >= s.bound) list(r, k, i, mass_at(k));
    });
  } else if (s.kind == kTopP) {
    const Bins bin(a, s.par, s.top);
    row.each([&](uint32_t k, int) {
      const u64 m = k ? mass_at(k) : 0;
      if (m) atomicAdd(&bins[kBins - 1 - bin(k)], m);
    });
    __syncthreads();
    for (int i = tid; i < kBins; i += 256)
      if (bins[i]) atomicAdd(&r.bins[i], bins[i]);
  } else {
    const u64 need = least(s.par.minp, a.bits);
    u64 sum = 0;
    row.each([&](uint32_t k, int) {
      const u64 m = k ? mass_at(k) : 0;
      sum += m >= need ? m : 0;
    });
    sum = wave_sum(sum);
    if (l == 0) r.sums[4 * b + w] = sum;
  }
}

__global__ void __launch_bounds__(kWide) k_split_bin(const DrawArgs a, SplitRow* rows) {
  __shared__ WideLds L;
  const long n = blockIdx.x;
  SplitRow& r = rows[n];
  const SplitState s(a, r, n);
  if (s.kind != kTopP) return;
  u64 all = 0;
  for (int i = threadIdx.x; i < kBins; i += kWide) {
    L.bins[i] = r.bins[i];
    all += r.bins[i];
  }
  const u64 want = (u64)ceil(s.par.p * (double)block_sum(L, all));
  int bin;
  u64 above;
  pick_bin(L, kBins, want, bin, above);
  if (threadIdx.x == 0) {
    r.want = want;
    r.above = above;
    r.bin = kBins - 1 - bin;
  }
}

template <typename T> __global__ void __launch_bounds__(256) k_split_border(const DrawArgs a, SplitRow* rows) {
  __shared__ double table[kTable];
  const long n = blockIdx.y;
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x;
  SplitRow& r = rows[n];
  const SplitState s(a, r, n);
  if (s.kind != kTopP) return;
  for (int i = tid; i < kTable; i += 256) table[i] = exp2((double)i / kTable);
  __syncthreads();
  const Row<T> row(a, n, 4 * b + w, kParts);
  const Bins bin(a, s.par, s.top);
  const int border = r.bin;
  const u64 need = least(s.par.minp, a.bits);
  u64 sum = 0;
  row.each([&](uint32_t k, int i) {
    const int at = k ? bin(k) : kBins;
    if (at > border) return;
    const u64 m = units(mass_of(k, s.top, s.par.c, table), a.bits);
    if (at == border) list(r, k, i, m);
    else sum += m >= need ? m : 0;
  });
  sum = wave_sum(sum);
  if (l == 0) r.sums[4 * b + w] = sum;
}

template <typename T> __global__ void __launch_bounds__(kWide) k_split_draw(const DrawArgs a, SplitRow* rows) {
  __shared__ WideLds L;
  __shared__ double table[kTable];
  __shared__ u64 sums[kParts];
  const long n = blockIdx.x;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  SplitRow& r = rows[n];
  const SplitState s(a, r, n);
  if (s.kind == kNone || s.kind == kGreedy) {
    if (tid == 0) {
      a.act[n] = s.kind == kNone ? -1 : r.greedy;
      if (a.logp) a.logp[n] = s.kind == kNone ? -INFINITY : 0.f;
    }
    return;
  }
  table[tid] = exp2((double)tid / kTable);
  const bool uses_list = s.kind == kTopK || s.kind == kTopP;
  if (s.kind == kFallBack || (uses_list && r.count > kList)) {
    draw_row<T>(L, table, a, n);
    return;
  }
  uint32_t thr = 1;
  int cut = a.A;
  u64 mine = 0, before = r.above;
  int rank = 0;
  if (uses_list) {
    if (tid == 0) L.count = r.count;
    if (tid < r.count) {
      mine = L.order[tid] = r.order[tid];
      L.mass[tid] = r.mass[tid];
    }
    __syncthreads();
    if (s.kind == kTopK) {
      before = 0;
      compare(L, mine, rank, before);
      cut_at(L, tid < L.count && rank == s.par.k - 1, mine, thr, cut);
      draw_listed(L, a, n, s.par, s.top, thr, cut);
      return;
    }
    compare(L, mine, rank, before);
  }
  if (tid < kParts) sums[tid] = r.sums[tid];
  const bool kept = s.kind == kTopP && tid < L.count && before < r.want;
  if (s.kind == kTopP) {
    const int of = __syncthreads_count(kept);
    cut_at(L, kept && rank == of - 1, mine, thr, cut);
  }
  __syncthreads();
  const u64 need = least(s.par.minp, a.bits);
  if (kept && L.mass[tid] >= need) atomicAdd(&sums[(int)(0xffffffffu - (uint32_t)mine) / Row<T>::size(a.A, kParts)], L.mass[tid]);
  __syncthreads();
  u64 total = 0, front = 0, part = 0;
  for (int i = 0; i < kParts; i++) total += sums[i];
  const u64 target = (u64)((double)s.par.u * (double)total);
  for (int i = 0; i < kParts; i++) {  // the part where the sum exceeds, for the first wavefront
    part = sums[i];
    if (part && (front + part > target || front + part == total)) {
      if (w == 0) {
        auto left_at = [&](uint32_t k, int e) {
          if (!k || !(k > thr || (k == thr && e <= cut))) return 0ull;
          const u64 m = units(mass_of(k, s.top, s.par.c, table), a.bits);
          return m >= need ? m : 0ull;
        };
        draw_in_part<T>(a, n, Row<T>(a, n, i, kParts), left_at, front, target, total, s.top, s.par.c);
      }
      return;
    }
    front += part;
  }
}

template <typename T> int draw_t(const DrawArgs& a, hipStream_t st) {
  const long blocks = (a.N + 3) / 4, most = 1L << 20;
  const unsigned n = (unsigned)(blocks < most ? blocks : most);
  if (a.A <= 64) k_draw_wave<T, 1><<<n, 256, 0, st>>>(a);
  else if (a.A <= 256) k_draw_wave<T, 4><<<n, 256, 0, st>>>(a);
  else if (a.A <= 1024) k_draw_wave<T, 16><<<n, 256, 0, st>>>(a);
  else if (draw_split(a.N, a.A)) {
    SplitRow* rows = (SplitRow*)scratch(kSlotDraw, (size_t)a.N * sizeof(SplitRow));
    if (!rows) return PH_ERR_NOMEM;
    const dim3 parts(kSplit, (unsigned)a.N);
    k_split_keys<T><<<parts, 256, 0, st>>>(a, rows);
    k_split_masses<T><<<parts, 256, 0, st>>>(a, rows);
    if (a.top_p) {
      k_split_bin<<<(unsigned)a.N, kWide, 0, st>>>(a, rows);
      k_split_border<T><<<parts, 256, 0, st>>>(a, rows);
    }
    k_split_draw<T><<<(unsigned)a.N, kWide, 0, st>>>(a, rows);
  } else {
    k_draw_wide<T><<<(unsigned)(a.N < most ? a.N : most), kWide, 0, st>>>(a);
  }
  PH_LAUNCH_CHECK();
  return PH_OK;
}

}  // namespace
}  // namespace ph

using namespace ph;

extern "C" int ph_sample_filtered(int dtype, const void* logits, long ld, size_t N, size_t A, const float* u,
                                  const float* temperature, const int* top_k, const float* top_p, const float* min_p, int* act,
                                  float* logp, void* stream) {
  PH_REQUIRE(dtype == PH_F32 || dtype == PH_BF16, "sample_filtered: dtype must be F32 or BF16");
  PH_REQUIRE(A >= 1 && A <= (1u << 20) && N <= (1u << 30), "sample_filtered: %zu rows of %zu entries", N, A);
  PH_REQUIRE(ld == 0 || ld >= (long)A, "sample_filtered: row stride %ld below %zu entries", ld, A);
  if (N == 0) return PH_OK;
  PH_REQUIRE(logits && u && act, "sample_filtered: logits, u or act missing");
  const long e = dtype == PH_BF16 ? 2 : 4;
  const Span x = {logits, (long)A * e, {(long)N, 1, 1}, {ld * e, 0, 0}}, outs[] = {flat(act, (long)N * 4), flat(logp, (long)N * 4)};
  const void* rows[] = {u, temperature, top_k, top_p, min_p};
  for (const Span& o : outs) {  // over a row's own number or parameter an output may lie: it is written when that has been read
    PH_REQUIRE(!meet(o, x), "sample_filtered: an output shares elements with the logits");
    for (const void* r : rows) PH_REQUIRE(o.p == r || !meet(o, flat(r, (long)N * 4)), "sample_filtered: an output lies across an input");
  }
  PH_REQUIRE(!meet(outs[0], outs[1]), "sample_filtered: act and logp share elements");
  DrawArgs a{};
  a.x = logits; a.ld = ld; a.N = (long)N; a.A = (int)A; a.u = u; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p;
  a.min_p = min_p; a.act = act; a.logp = logp;
  a.bits = 62;  // of a mass of 1, so that A of them fit 63 bits
  while (((size_t)1 << (62 - a.bits)) < A) a.bits--;
  if (a.bits > 51) a.bits = 51;
  return dtype == PH_BF16 ? draw_t<uint16_t>(a, as_stream(stream)) : draw_t<float>(a, as_stream(stream));
}
