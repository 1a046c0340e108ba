// Pages of keys and values in 8 bits: the layout that the kernels share.
//
// A page holds 16 tokens.  For every (page, KV head) there is one block of 2 x 16 x D codes (keys,
// then values), whole numbers from -127 to 127 held in a byte as q + 128, and four fp32 scales: keys
// of tokens 0-7 and 8-15, values of tokens 0-7 and 8-15.  A code q stands for q * scale.  The codes lie in the order in which the 32 lanes of a warp
// take them as operands of mma m16n8k16, so a lane's 16-byte loads need no shuffles and meet no
// bank conflicts; with lane = 4 g + c:
//   keys    row r = 8 h + g, column d = 16 j + 8 t1 + 2 c + t0:
//           byte (j / 2) * 512 + lane * 16 + ((j % 2) * 2 + h) * 4 + 2 t0 + t1
//   values  row r = 8 h + 2 c + t, column d = 16 k + 8 m + g:
//           byte (k / 2) * 512 + lane * 16 + ((k % 2) * 2 + h) * 4 + 2 t + m
// Either way a 32-bit word holds two operand registers: bytes 0 and 2, and bytes 1 and 3.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace lkv {

constexpr int kPageTokens = 16;
constexpr int kScalesPerBlock = 4;  // fp32: keys 0-7, keys 8-15, values 0-7, values 8-15

// Value scales below this are taken as this in the softmax's maximum: the sum of weights, times their reciprocals, stays
// finite for rows of 2^20 keys and more (2^15 * 2^90 * 2^20).  Blocks of zeros are such, beside scales of any size: their
// weights times the scale would be below fp32's least from scales of 2^51 on, so the sum takes them without it.
constexpr float kMinValueScale = 8.0779357e-28f;  // 2^-90
constexpr float kMinValueScaleLog2 = -90.f;

// Four codes as two pairs of f16: bytes 0 and 2 of w in lo, bytes 1 and 3 in hi.  Exact: the byte q + 128 under
// f16's 0x64 is 1024 + 128 + q.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4240), b = __byte_perm(w, 0x64646464u, 0x4341);
  const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace lkv
