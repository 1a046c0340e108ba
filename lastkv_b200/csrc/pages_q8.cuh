// Pages of keys and values in 8 bits: the layout that the kernels share.
//
// A page holds 16 tokens.  For every (page, KV head) there is one block of 2 x 16 x D int8 codes
// (keys, then values) and four fp32 scales: keys of tokens 0-7 and 8-15, values of tokens 0-7 and
// 8-15.  A code q stands for q * scale.  The codes lie in the order in which the 32 lanes of a warp
// take them as operands of mma m16n8k16, so a lane's 16-byte loads need no shuffles and meet no
// bank conflicts; with lane = 4 g + c:
//   keys    row r = 8 h + g, column d = 16 j + 8 t1 + 2 c + t0:
//           byte (j / 2) * 512 + lane * 16 + ((j % 2) * 2 + h) * 4 + 2 t0 + t1
//   values  row r = 8 h + 2 c + t, column d = 16 k + 8 m + g:
//           byte (k / 2) * 512 + lane * 16 + ((k % 2) * 2 + h) * 4 + 2 t + m
// Either way a 32-bit word holds two operand registers: bytes 0 and 2, and bytes 1 and 3.
#pragma once

#include "common.cuh"

namespace lkv {

constexpr int kPageTokens = 16;
constexpr int kScalesPerBlock = 4;  // fp32: keys 0-7, keys 8-15, values 0-7, values 8-15

// Two pairs of int8 codes as bf16 pairs: bytes 0 and 2 of w in lo, bytes 1 and 3 in hi.  Exact: with
// low = the code's seven low bits, 0x4300 | low is 128 + low and 0x4300 | sign bit is 128 or 256 in
// bf16, whose difference is the code.  Seven instructions for four codes.
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  constexpr uint32_t kOne = 0x43004300u;
  auto pair = [](uint32_t v) {
    const uint32_t a = (v & 0x007f007fu) | kOne, b = (v & 0x00800080u) | kOne;
    const __nv_bfloat162 d =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  };
  lo = pair(w);
  hi = pair(w >> 8);
}

}  // namespace lkv
