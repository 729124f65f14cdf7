// What the attention kernels share: LDS swizzles of the K and V tiles, the maximum over a wave's halves, transposed fragment reads.
#pragma once
#include "common.h"

namespace fdm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

template <int D>
struct Swz {
  static constexpr int CPR = D / 8;  // 16-byte chunks per row
  // K image: conflict-free ds_read_b128 for 16-lane groups of distinct rows
  static __device__ __forceinline__ int k(int row, int ch) {
    if constexpr (D == 128) return ch ^ (row & 15);
    else return ch ^ ((row >> 1) & 7);
  }
  // V image: conflict-free ds_read_b64_tr_b16 (4 consecutive keys x 64 B per 32-lane half)
  static __device__ __forceinline__ int v(int row, int ch) {
    if constexpr (D == 128) return ch ^ ((row & 3) << 2);
    else return ch ^ (((row >> 1) & 1) << 2);
  }
};

// max over the two 32-lane halves of a wave (the two halves of a query row's keys), identical in both halves afterwards.
// NOT `__builtin_amdgcn_permlane32_swap(x, x)` + fmaxf of the two results: hipcc 7.2 folds that to the first result alone (it takes the
// swap of a value with itself for the identity), i.e. every lane gets the LOWER half's maximum: harmless for the bf16 kernels' results (a
// missed fix-up only lets P grow, bf16 has the exponent range) but it defeats the lazy row reference for half of the keys, and with e4m3 P
// (fp8 P.V) a missed fix-up is a NaN.  (The spiked-key check of tools/micro/attn_bench shows it.)
// s_nop: VALU-written VGPR -> v_permlane32_swap needs a wait state that nothing pads inside asm.
__device__ __forceinline__ float cross_half_max(float m) {
  float a = m, b = m;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));     // a = (lower, lower), b = (upper, upper)
  return fmaxf(a, b);
}

__device__ __forceinline__ i32x4 tr_pair(const uint8_t* p0, const uint8_t* p1) {
  s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p0);
  s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p1);
  i32x2 lo = __builtin_bit_cast(i32x2, a), hi = __builtin_bit_cast(i32x2, b);
  i32x4 r;
  r[0] = lo[0]; r[1] = lo[1]; r[2] = hi[0]; r[3] = hi[1];
  return r;
}

}  // namespace fdm
