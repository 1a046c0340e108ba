// The packed 4-bit weight and its codes, shared by the kernels that read it (w4.cu, w4_tile.cu).
//
// Packed weight (lkv_w4_pack, laid out once): blocks of 64 output rows x 128 columns,
// the blocks of 64 rows contiguous along k.  A block is 4 sub-tiles of 16 rows x 128
// columns (1 KB each, in the order of the mma.sync A fragments) followed by its scales:
//   word (r, j, lane, i) at r * 1024 + j * 512 + lane * 16 + i * 4 holds
//     row 16 r + lane / 4 + 8 (i & 1), columns 32 (2 j + i / 2) + 8 (lane & 3) .. + 7,
//     byte b = code of column b (low half) and of column 4 + b (high half), two's complement
//   scale (gi, row 16 r + 8 h + g) at 4096 + 128 gi + 2 (8 g + 2 r + h), bf16
// so a warp reads a sub-tile with two 16-byte loads per lane, a lane's word holds eight
// neighbouring columns of one row, and a lane's eight scales of a group are one load.
// Rows and columns past the edge are zero.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace lkv {

constexpr int kTileRows = 64;
constexpr int kTileK = 128;
constexpr int kCodeBytes = kTileRows * kTileK / 2;

__host__ __device__ constexpr int block_bytes(int group) { return kCodeBytes + kTileRows * 2 * (kTileK / group); }

// Two of a word's codes (I = 0: columns 0, 2; 1: 4, 6; 2: 1, 3; 3: 5, 7) as exact bf16:
// 128 + (c + 8) by its mantissa bits, minus 136.
template <int I>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {
  const uint32_t m = ((w >> (4 * I)) & 0x000f000fu) ^ 0x43084308u;
  __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&m);
  v = __hsub2(v, __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<uint32_t*>(&v);
}

// More tokens than the skinny kernel takes well: tcgen05 tiles (w4_tile.cu).  LKV_ERR_UNSUPPORTED
// where the rows' alignment rules a TMA copy out.
bool w4_tile_aligned(const W4Args& a);
int w4_tile(const W4Args& a, int sms, cudaStream_t stream);

}  // namespace lkv
