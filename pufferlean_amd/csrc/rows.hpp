// Rows of a matrix in the registers of a few lanes, any width and alignment: what the normalisations share.
#pragma once
#include "common.hpp"

namespace ph {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// V consecutive elements at p as fp32: one 16-byte access for V = 8 (bf16) and V = 4 (fp32), else one element. AL: p is
// 16-byte aligned, and the row streams past the caches; rows of odd width start anywhere, which the hardware takes at
// element alignment, and share their lines with their neighbours.
template <typename T, int V, bool AL> __device__ __forceinline__ u32x4_t load16(const T* p) {
  u32x4_t r;
  if constexpr (AL) r = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
  else __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T, bool AL> __device__ __forceinline__ void store16(T* p, const u32x4_t& r) {
  if constexpr (AL) __builtin_nontemporal_store(r, reinterpret_cast<u32x4_t*>(p));
  else __builtin_memcpy(p, &r, 16);
}
template <int V, bool AL> __device__ __forceinline__ void load_v(const uint16_t* p, float* v) {
  if constexpr (V == 8) {
    const u32x4_t r = load16<uint16_t, V, AL>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __builtin_bit_cast(float, r[i] << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, r[i] & 0xffff0000u);
    }
  } else {
    v[0] = bf16_to_f32(*p);
  }
}
template <int V, bool AL> __device__ __forceinline__ void load_v(const float* p, float* v) {
  if constexpr (V == 4) {
    const u32x4_t r = load16<float, V, AL>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t u = r[i];  // a bit cast of the vector's element itself takes element 0
      v[i] = __builtin_bit_cast(float, u);
    }
  } else {
    v[0] = *p;
  }
}
template <int V, bool AL> __device__ __forceinline__ void store_v(uint16_t* p, const float* v) {
  if constexpr (V == 8) {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = bf16x2_rne(v[2 * i], v[2 * i + 1]);
    store16<uint16_t, AL>(p, r);
  } else {
    *p = bf16_rne(v[0]);
  }
}
template <int V, bool AL> __device__ __forceinline__ void store_v(float* p, const float* v) {
  if constexpr (V == 4) {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = __builtin_bit_cast(uint32_t, v[i]);
    store16<float, AL>(p, r);
  } else {
    *p = v[0];
  }
}

// The V columns that a lane holds in its access at column c of a row of C >= V: the last access of a row whose width is no
// multiple of V is moved back to the row's last V columns, of which it takes those from index `skip` on.
template <int V> struct Cols {
  int c, skip;
  bool in;
  __device__ __forceinline__ Cols(int at, int C) {
    in = at < C;
    c = V > 1 && at + V > C ? C - V : at;
    skip = at - c;
  }
  __device__ __forceinline__ bool has(int i) const { return in && i >= skip; }
};
// The access at k of row p, zero where it has no columns; and its store.
template <int V, bool AL, typename T>
__device__ __forceinline__ void get_cols(const Cols<V>& k, const T* p, float* v) {
#pragma unroll
  for (int i = 0; i < V; i++) v[i] = 0.f;
  if (k.in) load_v<V, AL>(p + k.c, v);
  if constexpr (V > 1 && !AL) {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = i >= k.skip ? v[i] : 0.f;
  }
}
template <int V, bool AL, typename T>
__device__ __forceinline__ void put_cols(const Cols<V>& k, T* p, const float* v) {
  if (!k.in) return;
  if (AL || k.skip == 0) {
    store_v<V, AL>(p + k.c, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
      if (i >= k.skip) store_v<1, false>(p + k.c + i, v + i);
  }
}

// The columns of w (or b) that a lane holds, 16 bytes at a time.
template <int V>
__device__ __forceinline__ void get_weights(const Cols<V>& k, const float* w, float none, float* v) {
#pragma unroll
  for (int i = 0; i < V; i++) v[i] = none;
  if (!w || !k.in) return;
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) load_v<4, false>(w + k.c + i, v + i);
  } else {
    v[0] = w[k.c];
  }
}

// dw, db = the partials' sums in a fixed order: 16 ranges of blocks per column, eight loads in flight each.
__global__ void __launch_bounds__(256) k_norm_fold(const float* __restrict__ part, int blocks, int C,
                                                   float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float sh[16][16];
  const int e = threadIdx.x & 15, z = threadIdx.x >> 4, col = blockIdx.x * 16 + e;
  const int per = (blocks + 15) / 16, end = min(blocks, (z + 1) * per);
  float s = 0.f;
  if (col < 2 * C) {
    int i = z * per;
    for (; i + 8 <= end; i += 8) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; q++) v[q] = part[(long)(i + q) * 2 * C + col];
#pragma unroll
      for (int q = 0; q < 8; q++) s += v[q];
    }
    for (; i < end; i++) s += part[(long)i * 2 * C + col];
  }
  sh[z][e] = s;
  __syncthreads();
  if (z || col >= 2 * C) return;
  for (int q = 1; q < 16; q++) s += sh[q][e];
  if (col < C) {
    if (dw) dw[col] = s;
  } else if (db) {
    db[col - C] = s;
  }
}

}  // namespace
}  // namespace ph
