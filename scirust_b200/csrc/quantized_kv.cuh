// Codes of the paged KV cache in 8 bits as numbers, and what its kernels check of a pool's layout.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace sb {
namespace kv8 {

// The larger magnitudes of two pairs in bf16, NaN above all, under some sign.
__device__ __forceinline__ uint32_t largest(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// Four codes as numbers.
template <bool E4M3>
__device__ __forceinline__ float4 from_codes(uint32_t w) {
  if constexpr (E4M3) {
    const float2 lo = __half22float2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffff), __NV_E4M3));
    const float2 hi = __half22float2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
  } else {
    // 2^23 + (code + 128) is a float whose last byte is that sum
    const uint32_t u = w ^ 0x80808080u;
    auto number = [u](uint32_t sel) { return __uint_as_float(__byte_perm(u, 0x4b000000u, sel)) - 8388736.f; };
    return make_float4(number(0x7440), number(0x7441), number(0x7442), number(0x7443));
  }
}

inline bool layout_ok(int Hkv, int dh, int n_blocks, int page, int block) {
  return Hkv > 0 && (dh == 64 || dh == 128) && n_blocks > 0 && page > 0 && (block == 8 || block == 16 || block == 32 || block == 64) &&
         page % block == 0;
}

}  // namespace kv8
}  // namespace sb
