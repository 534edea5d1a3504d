// Exchanges between the lanes of a wavefront by vector instructions: a sum over lanes through LDS permutations costs a
// hundred cycles and more a step.
#pragma once
#include <hip/hip_runtime.h>

namespace ph {

// The value of another lane of the same row of 16: lane ^ 1 (0xB1), lane ^ 2 (0x4E), lane ^ 7 (0x141), lane ^ 8 (0x128),
// lane ^ 15 (0x140).
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

// Sums of a and b over aligned groups of N lanes (8, 16, 32 or 64), in every lane of the group. All lanes of the groups are
// active.
template <int N> __device__ __forceinline__ void group_sum(float& a, float& b) {
  static_assert(N == 8 || N == 16 || N == 32 || N == 64, "group of lanes");
  a += dpp_mov<0xB1>(a);
  b += dpp_mov<0xB1>(b);
  a += dpp_mov<0x4E>(a);
  b += dpp_mov<0x4E>(b);
  a += dpp_mov<0x141>(a);
  b += dpp_mov<0x141>(b);
  if constexpr (N >= 16) {
    a += dpp_mov<0x140>(a);
    b += dpp_mov<0x140>(b);
  }
  if constexpr (N >= 32) {  // a register exchanged with its own copy: rows 0, 0, 2, 2 and 1, 1, 3, 3
    float a2 = a, b2 = b;
    swap16(a, a2, b, b2);
    a += a2;
    b += b2;
  }
  if constexpr (N >= 64) {
    float a2 = a, b2 = b;
    swap32(a, a2, b, b2);
    a += a2;
    b += b2;
  }
}
template <int N> __device__ __forceinline__ float group_sum(float a) {
  float b = 0.f;
  group_sum<N>(a, b);
  return a;
}

}  // namespace ph
