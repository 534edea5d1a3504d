// Draw of one entry per row of logits after temperature, top-k, top-p and min-p, from a given number u.
//
// What the filters leave is every entry above a threshold key, and of those at the threshold the ones up to an index:
// top-k's threshold is the k-th largest key, top-p's the one at which the mass of the larger ones reaches p of the total.
// Neither needs the row sorted: a key is a 32-bit number that orders like the logit, and the threshold is found digit by
// digit from the top, by how much (count, or mass) lies at and above each value of the digit. A whole row is then summed up in the
// order of its indices to where the sum exceeds u times the total.
//
// Masses are exp((l - max) / temperature) in 64-bit floating point, held as whole numbers of 2^-bits with as many bits as the
// sum of A of them has room for (45 at 131072 entries, 51 up to 2048): sums do not depend on their order, so the
// borders that u and p are compared with are the same however the row is split.
#include "common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

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
  double t, p;
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
  r.t = t > 0.f ? (double)t : 1.0;
  r.k = a.top_k && a.top_k[n] > 0 ? a.top_k[n] : a.A;
  r.greedy = t == 0.f || p <= 0.f;
  r.p = p < 1.f ? (double)p : 1.0;
  r.minp = m > 0.f ? (m < 1.f ? m : 1.f) : 0.f;
  r.u = a.u[n];
  return r;
}
// The mass of a key in units of 2^-bits; nothing below min_p.
__device__ __forceinline__ double mass_of(uint32_t key, uint32_t top, double t) {
  if (key == top) return 1.0;
  return exp(((double)logit_of(key) - (double)logit_of(top)) / t);
}
__device__ __forceinline__ u64 units(double e, int bits) { return (u64)__double2ll_rn(ldexp(e, bits)); }

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

// ---- rows in the registers of a wavefront ---------------------------------------------------------------------
// Entry 64 e + lane in register e; the digits are single bits, a count or sum over the wavefront each.
template <typename T, int E> __global__ void __launch_bounds__(256) k_draw_wave(const DrawArgs a) {
  const int l = threadIdx.x & 63;
  for (long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6); n < a.N; n += (long)gridDim.x * 4) {
    const T* row = (const T*)a.x + n * a.ld;
    uint32_t key[E], top = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int i = 64 * e + l;
      key[e] = i < a.A ? key_of(ldf(row + i)) : 0;
      top = key[e] > top ? key[e] : top;
    }
    top = wave_max(top);
    const Par par = par_of(a, n);
    int act = -1;
    float logp = -INFINITY;
    // the entries at `key` in the order of their indices: the index of the count-th (from 1)
    auto index_at = [&](uint32_t k, long count) {
      int cut = a.A;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const u64 on = __ballot(key[e] == k);
        const int c = __popcll(on);
        if (count > 0 && count <= c) {
          const u64 mine = on & ((2ull << l) - 1);
          const u64 at = __ballot(((on >> l) & 1) && __popcll(mine) == count);
          cut = 64 * e + __ffsll((unsigned long long)at) - 1;
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
      auto left = [&](int e) { return key[e] > thr || (key[e] == thr && 64 * e + l <= cut); };
      if (par.k < a.A) {
        uint32_t cur = 0;
        long at_least = 0;
        for (int bit = 31; bit >= 0; bit--) {
          const uint32_t c = cur | (1u << bit);
          long cnt = 0;
#pragma unroll
          for (int e = 0; e < E; e++) cnt += __popcll(__ballot(key[e] >= c));
          if (cnt >= par.k) {
            cur = c;
            at_least = cnt;
          }
        }
        if (cur) {  // else there are fewer than k
          thr = cur;
          if (at_least > par.k) {
            long above = 0;
#pragma unroll
            for (int e = 0; e < E; e++) above += __popcll(__ballot(key[e] > thr));
            cut = index_at(thr, par.k - above);
          }
        }
      }
      u64 m[E];
      u64 total = 0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        m[e] = key[e] && left(e) ? units(mass_of(key[e], top, par.t), a.bits) : 0;
        total += m[e];
      }
      if (par.p < 1.0) {
        total = wave_sum(total);
        const u64 want = (u64)ceil(par.p * (double)total);
        auto above = [&](uint32_t c) {  // mass of the keys over c
          u64 s = 0;
#pragma unroll
          for (int e = 0; e < E; e++) s += key[e] > c ? m[e] : 0;
          return wave_sum(s);
        };
        uint32_t cur = 0;
        for (int bit = 31; bit >= 0; bit--) {
          const uint32_t c = cur | (1u << bit);
          if (above(c) >= want) cur = c;
        }
        cur += 1;  // the smallest key with less than that above it
        const u64 each = units(mass_of(cur, top, par.t), a.bits), rest = want - above(cur);
        const u64 count = each ? (rest + each - 1) / each : 1;
        const int at = index_at(cur, (long)count);
        if (cur > thr) cut = a.A;
        thr = cur;
        cut = at < cut ? at : cut;
      }
      // in the order of the indices
      u64 sums[E];
      total = 0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const bool on = key[e] && left(e) && (par.minp == 0.f || mass_of(key[e], top, par.t) >= (double)par.minp);
        m[e] = on ? m[e] : 0;
        sums[e] = wave_sum(m[e]);
        total += sums[e];
      }
      const u64 target = (u64)((double)par.u * (double)total);  // a sum exceeds u total where it exceeds this
      u64 run = 0, got = 0;
      bool open = true;
#pragma unroll
      for (int e = 0; e < E; e++) {
        if (sums[e] == 0 || !open) continue;
        if (run + sums[e] > target || run + sums[e] == total) {
          const u64 at = run + wave_scan(m[e]);
          u64 hit = __ballot(m[e] > 0 && at > target);
          if (!hit) hit = 1ull << (63 - __clzll((long long)__ballot(m[e] > 0)));  // u rounded up to 1: the last
          const int lane = __ffsll((unsigned long long)hit) - 1;
          act = 64 * e + lane;
          got = __shfl(m[e], lane);
          open = false;
        }
        run += sums[e];
      }
      logp = (float)log((double)got / (double)total);
    }
    if (l == 0) {
      a.act[n] = act;
      if (a.logp) a.logp[n] = logp;
    }
  }
}

// ---- wide rows: a block each ----------------------------------------------------------------------------------
// Digits of 11, 11 and 10 bits, each by a histogram in LDS.
constexpr int kWide = 1024, kBins = 2048;

struct WideLds {
  u64 bins[kBins], wave[16], out[2];
  uint32_t key;
  int found;
};

// The largest bin b with sum(bins[b..]) >= want, in every thread: found, and above = sum(bins[b + 1 ..]). Every thread calls.
__device__ __forceinline__ void pick_bin(WideLds& L, int nbins, u64 want, int& bin, u64& above) {
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  __syncthreads();
  if (tid == 0) L.found = 0, L.out[0] = 0;
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
      L.out[0] = before;
    } else if (before + x0 + x1 >= want) {
      L.found = b0 - 1;
      L.out[0] = before + x0;
    }
  }
  __syncthreads();
  bin = L.found;
  above = L.out[0];
}

template <typename T> __global__ void __launch_bounds__(kWide) k_draw_wide(const DrawArgs a) {
  __shared__ WideLds L;
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  // the wavefront's part of the row, in whole tiles of 64 entries
  const int part = (a.A + 16 * 64 - 1) / (16 * 64) * 64, from = w * part < a.A ? w * part : a.A, to = from + part < a.A ? from + part : a.A;
  for (long n = blockIdx.x; n < a.N; n += gridDim.x) {
    const T* row = (const T*)a.x + n * a.ld;
    const Par par = par_of(a, n);
    auto key_at = [&](int i) { return key_of(ldf(row + i)); };
    __syncthreads();
    uint32_t top = 0;
    for (int i = tid; i < a.A; i += kWide) {
      const uint32_t k = key_at(i);
      top = k > top ? k : top;
    }
    top = wave_max(top);
    if (l == 0) L.wave[w] = top;
    __syncthreads();
    for (int i = 0; i < 16; i++) top = (uint32_t)L.wave[i] > top ? (uint32_t)L.wave[i] : top;
    if (top == 0) {
      if (tid == 0) {
        a.act[n] = -1;
        if (a.logp) a.logp[n] = -INFINITY;
      }
      continue;
    }
    // the index of the count-th entry (from 1) with this key, by the wavefronts' parts
    auto index_at = [&](uint32_t k, u64 count) {
      int c = 0;
      for (int i = from + l; i < from + part; i += 64) c += __popcll(__ballot(i < to && key_at(i) == k));
      __syncthreads();
      if (l == 0) L.wave[w] = (u64)c;
      if (tid == 0) L.found = a.A;
      __syncthreads();
      u64 before = 0;
      for (int i = 0; i < w; i++) before += L.wave[i];
      if (before < count && count <= before + c) {
        for (int i = from + l; i < from + part; i += 64) {
          const u64 on = __ballot(i < to && key_at(i) == k);
          const int here = __popcll(on);
          if (before < count && count <= before + here && ((on >> l) & 1) && before + __popcll(on & ((2ull << l) - 1)) == count)
            L.found = i;
          before += here;
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
      continue;
    }
    uint32_t thr = 1;
    int cut = a.A;
    auto mass_at = [&](uint32_t k, int i) {
      return k > thr || (k == thr && i <= cut) ? units(mass_of(k, top, par.t), a.bits) : 0ull;
    };
    // the threshold: the largest key at and above which there is `want` (entries, or mass), and what is wanted of those at it
    auto select = [&](bool mass, u64 want, u64& rest) {
      uint32_t key = 0;
      int have = 0;  // bits of the key that are known
      for (int d = 0; d < 3; d++) {
        const int bits = d < 2 ? 11 : 10, shift = 32 - have - bits;
        for (int i = tid; i < kBins; i += kWide) L.bins[i] = 0;
        __syncthreads();
        for (int i = tid; i < a.A; i += kWide) {
          const uint32_t k = key_at(i);
          if (!k || (have && (k >> (32 - have)) != key >> (32 - have))) continue;
          const u64 v = mass ? mass_at(k, i) : 1;
          if (v) atomicAdd(&L.bins[k >> shift & ((1u << bits) - 1)], v);
        }
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
    if (par.k < a.A) {
      int valid = 0;
      for (int i = tid; i < a.A; i += kWide) valid += key_at(i) != 0;
      const u64 v = wave_sum((u64)valid);
      __syncthreads();
      if (l == 0) L.wave[w] = v;
      __syncthreads();
      u64 all = 0;
      for (int i = 0; i < 16; i++) all += L.wave[i];
      if (all > (u64)par.k) {
        u64 rest;
        const uint32_t k = select(false, (u64)par.k, rest);
        cut = index_at(k, rest);
        thr = k;
      }
    }
    auto block_sum = [&](u64 v) {
      v = wave_sum(v);
      __syncthreads();
      if (l == 0) L.wave[w] = v;
      __syncthreads();
      u64 all = 0;
      for (int i = 0; i < 16; i++) all += L.wave[i];
      return all;
    };
    if (par.p < 1.0) {
      u64 s = 0;
      for (int i = tid; i < a.A; i += kWide) {
        const uint32_t k = key_at(i);
        if (k) s += mass_at(k, i);
      }
      const u64 want = (u64)ceil(par.p * (double)block_sum(s));
      u64 rest;
      const uint32_t k = select(true, want, rest);
      const u64 each = units(mass_of(k, top, par.t), a.bits), count = each ? (rest + each - 1) / each : 1;
      const int at = index_at(k, count);
      if (k > thr) cut = a.A;
      thr = k;
      cut = at < cut ? at : cut;
    }
    auto left_at = [&](uint32_t k, int i) {
      if (!k || !(k > thr || (k == thr && i <= cut))) return 0ull;
      const double e = mass_of(k, top, par.t);
      return e >= (double)par.minp ? units(e, a.bits) : 0ull;
    };
    u64 s = 0;
    for (int i = from + l; i < to; i += 64) s += left_at(key_at(i), i);
    const u64 mine = wave_sum(s);
    const u64 total = block_sum(s);  // L.wave: the wavefronts' sums
    u64 before = 0;
    for (int i = 0; i < w; i++) before += L.wave[i];
    const u64 target = (u64)((double)par.u * (double)total);
    if (mine && before <= target && (before + mine > target || before + mine == total)) {
      bool open = true;
      for (int i = from + l; i < from + part && open; i += 64) {
        const u64 m = i < to ? left_at(key_at(i), i) : 0;
        const u64 here = wave_sum(m);
        if (here && (before + here > target || before + here == total)) {
          const u64 at = before + wave_scan(m);
          u64 hit = __ballot(m > 0 && at > target);
          if (!hit) hit = 1ull << (63 - __clzll((long long)__ballot(m > 0)));
          if (l == __ffsll((unsigned long long)hit) - 1) {
            a.act[n] = i;
            if (a.logp) a.logp[n] = (float)log((double)m / (double)total);
          }
          open = false;
        }
        before += here;
      }
    }
  }
}

template <typename T> int draw_t(const DrawArgs& a, hipStream_t st) {
  const long blocks = (a.N + 3) / 4, most = 1L << 20;
  const unsigned n = (unsigned)(blocks < most ? blocks : most);
  if (a.A <= 64) k_draw_wave<T, 1><<<n, 256, 0, st>>>(a);
  else if (a.A <= 256) k_draw_wave<T, 4><<<n, 256, 0, st>>>(a);
  else if (a.A <= 1024) k_draw_wave<T, 16><<<n, 256, 0, st>>>(a);
  else k_draw_wide<T><<<(unsigned)(a.N < most ? a.N : most), kWide, 0, st>>>(a);
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
  DrawArgs a{};
  a.x = logits; a.ld = ld; a.N = (long)N; a.A = (int)A; a.u = u; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p;
  a.min_p = min_p; a.act = act; a.logp = logp;
  a.bits = 62;  // of a mass of 1, so that A of them fit 63 bits
  while (((size_t)1 << (62 - a.bits)) < A) a.bits--;
  if (a.bits > 51) a.bits = 51;
  return dtype == PH_BF16 ? draw_t<uint16_t>(a, as_stream(stream)) : draw_t<float>(a, as_stream(stream));
}
