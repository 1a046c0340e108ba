// The packed 4-bit weight and its codes, shared by the kernels that read it (w4.cu, w4_tile.cu).
//
// Packed weight (lkv_w4_pack, laid out once): blocks of 32 output rows x 128 columns; the
// four row blocks of 128 rows (the last ones may be fewer) lie side by side, then the next
// 128 columns, so a tile of 128 rows reads 128 columns with one copy.  A block is 2 sub-tiles of 16 rows x 128 columns (1 KB
// each, in the order of the mma.sync A fragments) followed by its scales:
//   word (r, j, lane, i) at r * 1024 + j * 512 + lane * 16 + i * 4 holds
//     row 16 r + lane / 4 + 8 (i & 1), columns 32 (2 j + i / 2) + 8 (lane & 3) .. + 7,
//     byte b = code of column b (low half) and of column 4 + b (high half), two's complement
//   scale (gi, row 16 r + 8 h + g) at 2048 + 64 gi + 2 (4 g + 2 r + h), bf16
// so a lane reads a sub-tile with two 16-byte loads, a word holds eight neighbouring columns
// of one row, a lane's four scales of a group are one load, and a block is one bulk copy.
// Rows and columns past the edge are zero.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace lkv {

constexpr int kTileRows = 32;
constexpr int kTileK = 128;
constexpr int kCodeBytes = kTileRows * kTileK / 2;

__host__ __device__ constexpr int block_bytes(int group) { return kCodeBytes + kTileRows * 2 * (kTileK / group); }

// First byte of block (rb, kb).
__host__ __device__ __forceinline__ int64_t block_offset(int64_t rb, int64_t kb, int kblocks, int row_blocks,
                                                         int group) {
  const int64_t first = rb & ~int64_t(3);
  const int64_t wide = row_blocks - first < 4 ? row_blocks - first : 4;
  return (first * kblocks + kb * wide + (rb - first)) * block_bytes(group);
}

// A condition that no value meets, which the compiler does not know.  A slot of shared memory
// that bulk copies refill may be released only once the values read from it have arrived in
// registers.  An mbarrier arrival or __syncwarp behind the loads does not see to that: loads
// whose results are used later were overtaken by the next copy, 64-byte pieces of which then
// stood in the block.  A vote on the loaded values waits for them in every lane.
struct Never {
  uint32_t a = 0, b = 1;
  __device__ __forceinline__ bool is(uint32_t v) const { return v == a && v == b; }
};

// Two of a word's codes (I = 0: columns 0, 2; 1: 4, 6; 2: 1, 3; 3: 5, 7) as exact bf16:
// 128 + (c + 8) by its mantissa bits, minus 136.
template <int I>
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w) {
  uint32_t m;  // (w & 0x000f000f) ^ 0x43084308 in one instruction (the compiler makes two of it)
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(m) : "r"(w >> (4 * I)), "r"(0x000f000fu), "r"(0x43084308u));
  __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&m);
  v = __hsub2(v, __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<uint32_t*>(&v);
}

// More tokens than the skinny kernel takes well: tcgen05 tiles (w4_tile.cu).  LKV_ERR_UNSUPPORTED
// where the rows' alignment rules a TMA copy out.
bool w4_tile_aligned(const W4Args& a);
int w4_tile(const W4Args& a, int sms, cudaStream_t stream);

}  // namespace lkv
