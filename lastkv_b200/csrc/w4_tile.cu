// Products with 4-bit weights for more than a few tokens, on tcgen05 (sm_100a).
//
// Tile: 128 output rows (the MMA's M side) x TN tokens (N side).  Per 128 bytes of k (128
// columns of int8 rows, 64 of bf16 rows) one stage of shared memory holds the A operand -
// the codes, expanded from 4 bits to int8 (16 c) or bf16 (c, exact) - and the B operand, the
// rows as they are, by TMA; both K-major, 128-byte swizzled.
//
// Group scales stay out of the operands: a group's MMAs sum into one of two or four TMEM buffers
// from zero (int32 or fp32), and the eight drain warps add each finished group into fp32
// registers, scaled by the weight's scale of the row and, for int8 rows, by the token's,
// while the tensor core sums the next groups into the other buffers.  So
// int8 x 4-bit group sums are exact and no weight is rounded, at the price of reading
// 128 x TN sums from TMEM per group, which is what bounds it: 2048 tokens x 28672 x 4096 in
// groups of 128 take 455 us with bf16 rows (1057 TFLOP/s, 0.63 of the measured bf16 peak) and
// 535 us with int8 rows (899 TOP/s), whose sums need a second multiply-add each (timed without
// it, and without the conversion, 410 us); in groups of 64 and 32 (4096 x 4096) 77 -> 113 ->
// 181 us and 85 -> 145 -> 263 us.  Weights s * c rounded to bf16 need no group sums (376 and
// 59 us), but are off by up to 2^-8 each.  Four drain warpgroups, a second expanding one,
// 32-column loads, loads one chunk ahead and waits with a suspend hint were no faster.
//
// Roles of the 512 threads (one CTA per SM, persistent over the tiles):
//   warp 0  rows by TMA                     warp 1     tcgen05.mma issue, TMEM
//   warp 2  the tokens' scales (int8 rows)  warp 3     codes, weight scales by bulk copies
//   warps 4-7  codes -> A tiles, weight scales -> their own slots     warps 8-15 drain, epilogue
// Where the tiles alone do not fill the GPU, k is split over the CTAs of a cluster, whose
// partial tiles meet in shared memory (added in split order).

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "tcgen05.cuh"
#include "w4.cuh"

namespace lkv {

namespace {

constexpr int kM = 128;
constexpr int kQuarters = kM / kTileRows;  // packed row blocks of a tile
constexpr int kDrainWgs = 2;
constexpr int kThreads = 256 + 128 * kDrainWgs;
constexpr int kKernelId = 13;
constexpr int kAStage = kM * 128;
constexpr int kMaxSplits = 8;
constexpr float kBias = 12582912.f;  // 1.5 * 2^23
constexpr int kPartRow = kM + 4;  // of a partial tile: 4 keeps the stores of neighbouring tokens off each other's banks

struct TileParams {
  const uint8_t* packed;
  const float* x_scale;
  int64_t x_scale_row;
  const __nv_bfloat16* bias;
  __nv_bfloat16* y;
  int64_t y_row;
  int tokens, n, k, kblocks, row_blocks, tok_tiles, tiles, splits;
  int* err;
  Never never;
};

// Ring depths: A stages (16 KB, filled in the CTA), B stages (TN x 128 bytes, from L2).
template <int TN>
__host__ __device__ constexpr int a_stages() {
  return TN == 256 ? 3 : 4;
}
template <int TN>
__host__ __device__ constexpr int b_stages() {
  return TN == 256 ? 4 : TN == 128 ? 6 : 8;
}

// 128-column blocks of packed weights (8 KB and the scales for the tile's 128 rows) in flight
template <int TN>
__host__ __device__ constexpr int code_slots() {
  return TN == 256 ? 3 : TN == 128 ? 4 : 8;
}

template <int G, int TN>
__host__ __device__ constexpr int ring_bytes() {
  return a_stages<TN>() * kAStage + b_stages<TN>() * TN * 128 + code_slots<TN>() * kQuarters * block_bytes(G);
}

// TMEM buffers of group sums: two 256-token tiles fill its 512 columns
template <int TN>
__host__ __device__ constexpr int d_buffers() {
  return TN == 256 ? 2 : 4;
}

// blocks of weight scales in flight: as many as the codes run ahead of the drain
template <int G, int TN>
__host__ __device__ constexpr int scale_slots() {
  return TN == 256 ? (G == 32 ? 4 : 8) : 16;
}
constexpr int kXsGroups = 4;  // groups of the tokens' scales per slot: one 16-byte load

template <bool INT8, int G, int TN>
struct Shared {
  uint64_t a_full[a_stages<TN>()], a_empty[a_stages<TN>()];
  uint64_t b_full[b_stages<TN>()], b_empty[b_stages<TN>()];
  uint64_t d_full[d_buffers<TN>()], d_empty[d_buffers<TN>()];
  uint64_t done;
  uint64_t c_full[code_slots<TN>()], c_empty[code_slots<TN>()];
  uint64_t ws_full[scale_slots<G, TN>()], ws_empty[scale_slots<G, TN>()];
  uint64_t xs_full[2], xs_empty[2];
  uint32_t tmem;
  alignas(16) uint8_t ws[scale_slots<G, TN>()][kQuarters][kTileRows * 2 * (kTileK / G)];  // the weight's scales of a 128-column block
  alignas(16) float xs[INT8 ? 2 : 1][kXsGroups][INT8 ? TN : 4];  // the tokens' scales
};

template <bool INT8, int G, int TN>
constexpr int smem_bytes() {
  return 1024 + ring_bytes<G, TN>() + (int)sizeof(Shared<INT8, G, TN>);
}

template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void st_shared8(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// 1.5 * 2^23 + v for an int32 |v| < 2^22 (128 x 127 x 128 < 2^21 here), exactly: the integer sum
// of v and the bits of 1.5 * 2^23, which masking and flipping bit 22 give for either sign.
// (A logic instruction: the add goes to the fp32 pipe, which the drain fills already, and a
// conversion runs at an eighth of their rate.)
__device__ __forceinline__ float int_bits(uint32_t v) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(v), "r"(0x007fffffu), "r"(0x4b400000u));
  return __uint_as_float(r);
}

template <bool INT8, int G, int TN>
__global__ void __launch_bounds__(kThreads, 1)
    w4_tile_kernel(const __grid_constant__ CUtensorMap tmx, const TileParams p) {
  constexpr int kWsSlots = scale_slots<G, TN>();
  constexpr int SA = a_stages<TN>(), SB = b_stages<TN>(), C = code_slots<TN>(), kBStage = TN * 128, ND = d_buffers<TN>();
  constexpr int kSpb = INT8 ? 1 : 2;               // stages per 128-column block
  constexpr int kMpg = INT8 ? G / 32 : G / 16;     // MMAs per group
  constexpr int kGpb = kTileK / G;                 // groups per block
  constexpr int kCols = TN / kDrainWgs;            // tokens of one drain warpgroup
  constexpr uint32_t kIdesc = INT8 ? umma_idesc_s8(kM, TN) : umma_idesc_bf16(kM, TN, 0, 0);
  constexpr uint32_t kTmemCols = ND * TN;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Sh = Shared<INT8, G, TN>;
  uint8_t* b_ring = smem + SA * kAStage;
  uint8_t* codes = b_ring + SB * kBStage;  // [C][kQuarters][block_bytes(G)]
  Sh* sh = reinterpret_cast<Sh*>(smem + ring_bytes<G, TN>());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.y;
  const int kb0 = (int)((int64_t)p.kblocks * split / p.splits);
  const int kb1 = (int)((int64_t)p.kblocks * (split + 1) / p.splits);
  const int nkb = kb1 - kb0;
  pdl_launch_dependents();

  if (threadIdx.x == 0) {
    for (int s = 0; s < SA; ++s) {
      mbar_init(&sh->a_full[s], 4);
      mbar_init(&sh->a_empty[s], 1);
    }
    for (int s = 0; s < SB; ++s) {
      mbar_init(&sh->b_full[s], 1);
      mbar_init(&sh->b_empty[s], 1);
    }
    for (int b = 0; b < ND; ++b) {
      mbar_init(&sh->d_full[b], 1);
      mbar_init(&sh->d_empty[b], 4 * kDrainWgs);
    }
    mbar_init(&sh->done, 1);
    for (int b = 0; b < C; ++b) {
      mbar_init(&sh->c_full[b], 1);
      mbar_init(&sh->c_empty[b], 4);
    }
    for (int b = 0; b < kWsSlots; ++b) {
      mbar_init(&sh->ws_full[b], 4);
      mbar_init(&sh->ws_empty[b], 4 * kDrainWgs);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh->xs_full[b], 1);
      mbar_init(&sh->xs_empty[b], 4 * kDrainWgs);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sh->tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;

  if (warp < 4) {
    regs_dec<40>();
    if (warp == 0) {
      if (lane == 0) {
        // ------------------------------------------------------------ rows by TMA
        tma_prefetch_desc(&tmx);
        pdl_wait();
        uint32_t it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
          const int tok0 = tile % p.tok_tiles * TN;
          for (int i = 0; i < nkb * kSpb; ++i, ++it) {
            const int s = it % SB;
            ok = mbar_wait(&sh->b_empty[s], ((it / SB) & 1) ^ 1);
            if (!ok) break;
            mbar_arrive_expect_tx(&sh->b_full[s], kBStage);
            tma_load_2d(b_ring + s * kBStage, &tmx, &sh->b_full[s], (kb0 * kSpb + i) * (INT8 ? 128 : 64), tok0);
          }
        }
        if (!ok) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, (int)it);
        // No copy may still be in flight when the CTA leaves, whichever warp's wait gave up.
        for (uint32_t i = it > SB ? it - SB : 0; i < it; ++i) mbar_wait(&sh->b_full[i % SB], (i / SB) & 1);
      }
    } else if (warp == 1) {
      // -------------------------------------------------------------- MMA issue
      // One MMA of a 256-token tile takes 128 cycles, so the loop is kept short: stages and
      // phases are counted, descriptors are additions to two bases, and the MMAs of a stage
      // (or of a group inside one) go out together.
      constexpr int kRun = kMpg < 4 ? kMpg : 4;        // MMAs between two waits
      constexpr int kStagesPerGroup = kMpg / kRun;     // 1, or 2 (bf16 rows in groups of 128)
      const uint64_t desc_a = umma_sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t desc_b = umma_sdesc_sw128(smem_u32(b_ring), 16, 1024);
      uint32_t it = 0, sa = 0, sb = 0, pa = 0, pb = 0, buf = 0, pd = 1, in_group = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
        for (int i = 0; i < nkb * kSpb; ++i, ++it) {
          ok = mbar_wait(&sh->a_full[sa], pa) && mbar_wait(&sh->b_full[sb], pb);
          const uint64_t da = desc_a + sa * (kAStage >> 4), db = desc_b + sb * (kBStage >> 4);
#pragma unroll
          for (int r = 0; r < 4 / kRun; ++r) {
            if (in_group == 0) ok = ok && mbar_wait(&sh->d_empty[buf], pd);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const bool last = in_group == kStagesPerGroup - 1;
            if (elect_one()) {
              const uint32_t d = tmem + buf * TN;
#pragma unroll
              for (int m = 0; m < kRun; ++m) {
                const int at = 2 * (r * kRun + m);  // 32 bytes of k, in descriptor units
                if (INT8)
                  umma_s8_ss(d, da + at, db + at, kIdesc, m > 0 || in_group > 0);
                else
                  umma_bf16_ss(d, da + at, db + at, kIdesc, m > 0 || in_group > 0);
              }
              if (r == 4 / kRun - 1) {
                umma_commit(&sh->a_empty[sa]);
                umma_commit(&sh->b_empty[sb]);
              }
              if (last) umma_commit(&sh->d_full[buf]);
            }
            __syncwarp();
            if (last) {
              in_group = 0;
              if (++buf == ND) buf = 0, pd ^= 1;
            } else {
              ++in_group;
            }
          }
          if (!ok) break;
          if (++sa == SA) sa = 0, pa ^= 1;
          if (++sb == SB) sb = 0, pb ^= 1;
        }
      }
      if (!ok && lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 1000000 + (int)it);
      if (elect_one()) umma_commit(&sh->done);
      __syncwarp();
      mbar_wait(&sh->done, 0);  // no MMA may still be in flight when TMEM is freed
    } else if (warp == 3) {
      // -------------------------------------------------------------- packed weights by bulk copies
      if (lane == 0) {  // before the previous kernel has finished: the weights do not depend on it
        uint32_t blk = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
          const int rb = tile / p.tok_tiles * kQuarters, quarters = min(kQuarters, p.row_blocks - rb);
          const uint32_t bytes = quarters * block_bytes(G);
          const uint8_t* src = p.packed + block_offset(rb, kb0, p.kblocks, p.row_blocks, G);
          for (int kb = 0; kb < nkb; ++kb, ++blk, src += bytes) {
            const int b = blk % C;
            ok = mbar_wait(&sh->c_empty[b], ((blk / C) & 1) ^ 1);
            if (!ok) break;
            mbar_arrive_expect_tx(&sh->c_full[b], bytes);
            bulk_load(codes + b * kQuarters * block_bytes(G), src, bytes, &sh->c_full[b]);
          }
        }
        if (!ok) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 5000000 + (int)blk);
        for (uint32_t i = blk > C ? blk - C : 0; i < blk; ++i) mbar_wait(&sh->c_full[i % C], (i / C) & 1);
      }
    } else if (INT8) {
      // -------------------------------------------------------------- the tokens' scales, transposed
      pdl_wait();
      const int groups = (p.k + G - 1) / G, g0 = kb0 * kGpb, g1 = kb1 * kGpb;
      const bool wide = (reinterpret_cast<uintptr_t>(p.x_scale) & 15) == 0 && p.x_scale_row % 4 == 0 && g0 % 4 == 0;
      uint32_t slot = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
        const int tok0 = tile % p.tok_tiles * TN;
        for (int gr = g0; ok && gr < g1; gr += kXsGroups, ++slot) {
          const int b = slot & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh->xs_empty[b], ((slot >> 1) & 1) ^ 1));
          if (!ok) break;
          for (int c = lane; c < TN; c += 32) {
            float v[kXsGroups];
            const float* src = p.x_scale + (int64_t)(tok0 + c) * p.x_scale_row + gr;
            if (tok0 + c < p.tokens && wide && gr + kXsGroups <= groups) {
              const float4 q = *reinterpret_cast<const float4*>(src);
              v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
            } else {
#pragma unroll
              for (int e = 0; e < kXsGroups; ++e) v[e] = tok0 + c < p.tokens && gr + e < groups ? src[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < kXsGroups; ++e) sh->xs[b][e][c] = v[e];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->xs_full[b]);
        }
      }
      if (!ok && lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 4000000 + (int)slot);
    }
  } else if (warp < 8) {
    // ---------------------------------------------------------------- codes -> A tiles
    // the block launches with 128 registers a thread: 40 + 88 + 2 x 192 = 4 x 128
    regs_dec<88>();
    constexpr int kN = INT8 ? 4 : 2;  // 16-byte pieces (rows g and g + 8 of a sub-tile, two 32-column steps) per lane
    // Piece of lane 4 g + t.  A phase of eight lanes reads all eight 16-byte banks of its 128
    // bytes (t and the parity of g) and stores to all eight swizzled chunks (chunk ^ g): the
    // rows of a phase are g and g ^ 5; phases in the order 0, 2, 1, 3 also keep the 8-byte
    // stores of half a warp apart.
    const int w = warp - 4, t = lane & 3, q3 = lane >> 3;
    const int g = ((q3 & 1) << 1 | q3 >> 1) ^ ((lane & 4) ? 5 : 0);
    uint32_t blk = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      const int quarters = min(kQuarters, p.row_blocks - tile / p.tok_tiles * kQuarters);
      for (int kb = 0; ok && kb < nkb; ++kb, ++blk) {
        const int b = blk % C, e = blk % kWsSlots;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->c_full[b], (blk / C) & 1) &&
                                         mbar_wait(&sh->ws_empty[e], ((blk / kWsSlots) & 1) ^ 1));
        if (!ok) break;
        const uint8_t* src = codes + (b * kQuarters + w) * block_bytes(G);
        // the row block's scales, for the drain
        for (int i = lane; i < kGpb * 16; i += 32)
          reinterpret_cast<uint32_t*>(sh->ws[e][w])[i] = ld_shared4(src + kCodeBytes + 4 * i);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->ws_full[e]);
        uint4 v[kSpb][kN];  // the whole block at once: 2048 bf16 rows x 4096 x 4096 71.4 us, a stage at a time 73.3
#pragma unroll
        for (int i = 0; i < kSpb; ++i)
#pragma unroll
          for (int q = 0; q < kN; ++q) {
            // warp w expands row block w: int8 pieces (r, j), bf16 pieces r, j from the stage
            const int r = INT8 ? q >> 1 : q, j = INT8 ? q & 1 : i;
            v[i][q] = w < quarters ? ld_shared16(src + r * 1024 + j * 512 + (4 * g + t) * 16) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
        for (int i = 0; i < kSpb; ++i) {
          const uint32_t it = blk * kSpb + i;
          const int s = it % SA;
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&sh->a_empty[s], ((it / SA) & 1) ^ 1));
          if (!ok) break;
          const uint32_t a = smem_u32(smem + s * kAStage);
#pragma unroll
          for (int q = 0; q < kN; ++q) {
            const int r = INT8 ? q >> 1 : q, j = INT8 ? q & 1 : 0;
            const uint32_t words[4] = {v[i][q].x, v[i][q].y, v[i][q].z, v[i][q].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t row = a + (w * kTileRows + 16 * r + 8 * (e & 1) + g) * 128;
              const uint32_t u = words[e];
              if (INT8) {
                const int chunk = 2 * (2 * j + (e >> 1)) + (t >> 1);
                st_shared8(row + ((chunk ^ g) << 4) + 8 * (t & 1), u << 4 & 0xf0f0f0f0u, u & 0xf0f0f0f0u);
              } else {
                const uint32_t c02 = codes_bf16<0>(u), c46 = codes_bf16<1>(u), c13 = codes_bf16<2>(u),
                               c57 = codes_bf16<3>(u);
                const int chunk = 4 * (e >> 1) + t;
                st_shared16(row + ((chunk ^ g) << 4), __byte_perm(c02, c13, 0x5410), __byte_perm(c02, c13, 0x7632),
                            __byte_perm(c46, c57, 0x5410), __byte_perm(c46, c57, 0x7632));
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sh->a_full[s]);
            // Not before the stores above, which need the loaded values: an arrival right after
            // the loads lets the next copy overwrite the block before they have read it.
            if (i == kSpb - 1) mbar_arrive(&sh->c_empty[b]);
          }
        }
      }
    }
    if (!ok && lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 2000000 + (int)blk);
  } else {
    // ---------------------------------------------------------------- drain, epilogue
    regs_inc<192>();
    // A lane holds, of each 8 tokens, two neighbours (2 q, 2 q + 1) in four rows (g, + 8, + 16,
    // + 24 of the warp's 32): a group's token scales are one 8-byte load for eight sums, where
    // a lane per row would need one for two and wait for shared memory.
    const int wg = (warp - 8) >> 2, sub = warp & 3, g = lane >> 2, q = lane & 3;
    const uint32_t lanes = (uint32_t)(sub * 32) << 16;
    uint32_t grp = 0, blk = 0, slot = 0;
    bool ok = true;
    pdl_wait();  // before any global write
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      const int tok0 = tile % p.tok_tiles * TN + wg * kCols;
      const int row0 = (tile / p.tok_tiles) * kM + sub * kTileRows;
      const bool live = row0 < p.row_blocks * kTileRows;
      float2 acc[2][kCols / 8][2];  // [16 rows][8 tokens][8 rows]
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < kCols / 8; ++c) acc[h][c][0] = acc[h][c][1] = make_float2(0.f, 0.f);
      int gt = 0;  // group of this tile's range
      for (int kb = 0; ok && kb < nkb; ++kb, ++blk) {
        const int b = blk % kWsSlots;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->ws_full[b], (blk / kWsSlots) & 1));
        if (!ok) break;
#pragma unroll 1
        for (int gi = 0; gi < kGpb; ++gi, ++gt) {
          const int buf = grp % ND;
          // scales of rows 16 h + 8 e + g at 2 (4 g + 2 h + e); int8 codes stand at 16 c.  With w such a scale
          // (8 bits) over 16, 1.5 * 2^23 w is exact too, so (1.5 * 2^23 + sum) w - 1.5 * 2^23 w is sum * w,
          // rounded once; the token's scale, with all its bits, multiplies that.
          const uint2 w4 = live ? ld_shared8(&sh->ws[b][sub][gi * 64 + g * 8]) : make_uint2(0, 0);
          constexpr float kUnit = INT8 ? 0.0625f : 1.f;
          const float ws[2][2] = {{bf16_lo(w4.x) * kUnit, bf16_hi(w4.x) * kUnit},
                                  {bf16_lo(w4.y) * kUnit, bf16_hi(w4.y) * kUnit}};
          const float* xs = &sh->xs[INT8 ? slot & 1 : 0][gt % kXsGroups][INT8 ? wg * kCols : 0] + 2 * q;
          if (INT8 && gt % kXsGroups == 0) ok = mbar_wait(&sh->xs_full[slot & 1], (slot >> 1) & 1);
          ok = ok && mbar_wait(&sh->d_full[buf], (grp / ND) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t at = tmem + lanes + buf * TN + wg * kCols;
          uint32_t u[2][8];
          auto load = [&](int c0) {
            tmem_ld_16x16(at + c0, u[0]);
            tmem_ld_16x16(at + (16u << 16) + c0, u[1]);
          };
          load(0);  // before the vote: 128 tokens x 28672 x 4096 48.9 us, 51.5 behind it
          // From about 2^104 on those products leave fp32's range: such a warp converts its sums first.
          const bool far = INT8 && __any_sync(0xffffffffu, fmaxf(fmaxf(fabsf(ws[0][0]), fabsf(ws[0][1])),
                                                                 fmaxf(fabsf(ws[1][0]), fabsf(ws[1][1]))) >= 0x1p100f);
          auto drain = [&](auto converts) {
            constexpr bool kConverts = decltype(converts)::value;
#pragma unroll
            for (int c0 = 0; c0 < kCols; c0 += 16) {
              if (c0 > 0) load(c0);
              tmem_wait_ld16(u);
              if (c0 + 16 == kCols) {  // the buffer is read: the tensor core may sum the next group but one
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->d_empty[buf]);
              }
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float2 x = make_float2(1.f, 1.f);
                if (INT8) {
                  const uint2 ux = ld_shared8(xs + c0 + 8 * c);
                  x = make_float2(__uint_as_float(ux.x), __uint_as_float(ux.y));
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const uint32_t lo = u[h][4 * c + 2 * e], hi = u[h][4 * c + 2 * e + 1];
                    const float w = ws[h][e];
                    float2& a = acc[h][c0 / 8 + c][e];
                    if (!INT8) {
                      a = __ffma2_rn(make_float2(__uint_as_float(lo), __uint_as_float(hi)), make_float2(w, w), a);
                    } else if (kConverts) {
                      a.x = fmaf(int_bits(lo) - kBias, w * x.x, a.x);
                      a.y = fmaf(int_bits(hi) - kBias, w * x.y, a.y);
                    } else {
                      const float2 v = __ffma2_rn(make_float2(int_bits(lo), int_bits(hi)), make_float2(w, w),
                                                  make_float2(-kBias * w, -kBias * w));
                      a = __ffma2_rn(v, x, a);
                    }
                  }
              }
            }
          };
          if (far)
            drain(std::true_type{});
          else
            drain(std::false_type{});
          ++grp;
          if (INT8 && (gt % kXsGroups == kXsGroups - 1 || gt == nkb * kGpb - 1)) {
            // the vote needs the last sums, and so the scales, in registers (see Never)
            if (!__any_sync(0xffffffffu, p.never.is(__float_as_uint(acc[1][kCols / 8 - 1][1].x))) && lane == 0)
              mbar_arrive(&sh->xs_empty[slot & 1]);
            ++slot;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->ws_empty[b]);
      }
      if (!ok) break;
      if (p.splits == 1) {
        // 8 rows x 8 tokens at a time through a register transpose: a lane then stores two
        // neighbouring rows of one token
        const bool words = ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)(p.y_row * 2)) & 3) == 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = row0 + 16 * h + 8 * e;
            const float bias = p.bias && r + g < p.n ? __bfloat162float(p.bias[r + g]) : 0.f;
            const int f = r + 2 * q;
#pragma unroll
            for (int c = 0; c < kCols / 8; ++c) {
              const uint32_t v = movmatrix_trans(pack_bf16(acc[h][c][e].x + bias, acc[h][c][e].y + bias));
              const int tok = tok0 + 8 * c + g;
              if (tok >= p.tokens) continue;
              __nv_bfloat16* y = p.y + (int64_t)tok * p.y_row + f;
              if (words && f + 1 < p.n) {
                *reinterpret_cast<uint32_t*>(y) = v;
              } else {
                if (f < p.n) y[0] = __ushort_as_bfloat16((unsigned short)v);
                if (f + 1 < p.n) y[1] = __ushort_as_bfloat16((unsigned short)(v >> 16));
              }
            }
          }
      } else {
        // one tile per cluster: every stage has been consumed, their memory takes the partial [token][row]
        float* part = reinterpret_cast<float*>(smem) + (wg * kCols + 2 * q) * kPartRow + sub * kTileRows + g;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < kCols / 8; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              part[8 * c * kPartRow + 16 * h + 8 * e] = acc[h][c][e].x;
              part[(8 * c + 1) * kPartRow + 16 * h + 8 * e] = acc[h][c][e].y;
            }
      }
    }
    if (!ok && lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 3000000 + (int)grp);
  }

  __syncwarp();
  if (p.splits > 1) {
    cluster_sync_all();  // every split has published its partial
    const int tile = blockIdx.x;
    const int tok0 = tile % p.tok_tiles * TN, row0 = tile / p.tok_tiles * kM;
    const bool words = ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)(p.y_row * 2)) & 3) == 0;
    const uint32_t base = smem_u32(smem);
    // A warp takes a token, a lane four rows of it: 16-byte loads, the splits' in flight together.
    // (4-byte loads: 256 bf16 rows x 6144 x 4096, two splits, 29.5 against 23.4 us.)
    constexpr int kWarps = kThreads / 32;
    const int tokens = min(TN, p.tokens - tok0), r = row0 + 4 * lane;
#pragma unroll 1
    for (int t = (int)cluster_rank() * kWarps + warp; t < tokens; t += p.splits * kWarps) {
      const uint32_t at = (uint32_t)(t * kPartRow + 4 * lane) * 4;
      float4 v[kMaxSplits];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s)
        v[s] = s < p.splits ? dsmem_ld4(dsmem_map(base, s) + at) : make_float4(0.f, 0.f, 0.f, 0.f);
      float sum[4] = {};
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) {
        sum[0] += v[s].x;
        sum[1] += v[s].y;
        sum[2] += v[s].z;
        sum[3] += v[s].w;
      }
      __nv_bfloat16* y = p.y + (int64_t)(tok0 + t) * p.y_row + r;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (p.bias && r + e < p.n) sum[e] += __bfloat162float(p.bias[r + e]);
      if (words && r + 3 < p.n) {
        reinterpret_cast<uint32_t*>(y)[0] = pack_bf16(sum[0], sum[1]);
        reinterpret_cast<uint32_t*>(y)[1] = pack_bf16(sum[2], sum[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r + e < p.n) y[e] = __float2bfloat16_rn(sum[e]);
      }
    }
    cluster_sync_all();  // the partials stay readable until every CTA has read them
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <bool INT8, int G, int TN>
int launch(const CUtensorMap& map, const TileParams& p, int sms, cudaStream_t stream) {
  static_assert(smem_bytes<INT8, G, TN>() <= 227 * 1024, "shared memory of a CTA");
  static_assert(TN * kPartRow * 4 <= ring_bytes<G, TN>(), "partial tile");
  static std::once_flag once[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LKV_ERR_CUDA;
  static cudaError_t set[64];
  std::call_once(once[dev], [&] {
    set[dev] = cudaFuncSetAttribute(w4_tile_kernel<INT8, G, TN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    smem_bytes<INT8, G, TN>());
  });
  if (set[dev] != cudaSuccess) return LKV_ERR_CUDA;
  const dim3 grid(std::min(p.tiles, std::max(1, sms / p.splits)), p.splits);
  return launch_pdl_cluster(w4_tile_kernel<INT8, G, TN>, grid, dim3(kThreads), smem_bytes<INT8, G, TN>(), stream,
                            dim3(1, p.splits, 1), map, p) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

template <bool INT8, int G>
int by_tokens(int tn, const CUtensorMap& map, const TileParams& p, int sms, cudaStream_t stream) {
  switch (tn) {
    case 64: return launch<INT8, G, 64>(map, p, sms, stream);
    case 128: return launch<INT8, G, 128>(map, p, sms, stream);
    default: return launch<INT8, G, 256>(map, p, sms, stream);
  }
}

}  // namespace

bool w4_tile_aligned(const W4Args& a) {
  const int elem = a.x_scale ? 1 : 2;
  return (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (a.x_row * elem) % 16 == 0;
}

int w4_tile(const W4Args& a, int sms, cudaStream_t stream) {
  const bool int8 = a.x_scale != nullptr;
  TileParams p{};
  p.packed = static_cast<const uint8_t*>(a.packed);
  p.x_scale = a.x_scale;
  p.x_scale_row = a.x_scale_row;
  p.bias = static_cast<const __nv_bfloat16*>(a.bias);
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.y_row = a.y_row;
  p.tokens = (int)a.tokens;
  p.n = (int)a.n;
  p.k = (int)a.k;
  p.kblocks = (int)((a.k + kTileK - 1) / kTileK);
  p.row_blocks = (int)((a.n + kTileRows - 1) / kTileRows);
  p.err = a.error_word;
  const int64_t row_tiles = (a.n + kM - 1) / kM;
  auto tiles = [&](int tn) { return row_tiles * ((a.tokens + tn - 1) / tn); };
  // A power of two of splits, while every CTA still has an SM and two blocks of k.  (Clusters that
  // the SMs' grouping leaves no room for run after the others; none waits for another.)
  auto splits = [&](int tn) {
    int s = 1;
    while (s < kMaxSplits && tiles(tn) * s * 2 <= sms && p.kblocks >= s * 4) s *= 2;
    return s;
  };
  // Tokens of a tile: 256 take 1.85 (int8) or 1.35 (bf16) times a 128-token tile's time in groups of
  // 128 (groups of 32: 1.73 and 1.86), which the rounds of tiles over the SMs may cost.  256 against 128, int8 / bf16 rows: 2048 tokens x 28672
  // x 4096 (13 against 25 rounds) 540 / 460 against 561 / 670 us; 1024 x 6144 (2, 3) 86 / 73 against
  // 71 / 85 us; 384 x 6144 (1, 1) 45 / 38 against 26 / 31 us; 512 x 28672 (4, 7) 168 / 143 against
  // 159 / 191 us.
  auto rounds = [&](int tn) { return (double)((tiles(tn) + sms - 1) / sms) / splits(tn); };
  const int tn = a.tokens <= 64                                                         ? 64
                 : a.tokens <= 128 || rounds(128) < rounds(256) * (int8 ? 1.85 : 1.35) ? 128
                                                                                        : 256;
  if (tiles(tn) > 0x7fffffff) return LKV_ERR_UNSUPPORTED;
  p.tok_tiles = (int)((a.tokens + tn - 1) / tn);
  p.tiles = (int)tiles(tn);
  p.splits = splits(tn);
  CUtensorMap map;
  const int st = int8 ? make_matrix_tensor_map_s8(&map, a.x, a.tokens, a.k, a.x_row, tn)
                      : make_matrix_tensor_map(&map, a.x, a.tokens, a.k, a.x_row, tn);
  if (st != LKV_OK) return st;
  if (int8)
    return a.group == 32   ? by_tokens<true, 32>(tn, map, p, sms, stream)
           : a.group == 64 ? by_tokens<true, 64>(tn, map, p, sms, stream)
                           : by_tokens<true, 128>(tn, map, p, sms, stream);
  return a.group == 32   ? by_tokens<false, 32>(tn, map, p, sms, stream)
         : a.group == 64 ? by_tokens<false, 64>(tn, map, p, sms, stream)
                         : by_tokens<false, 128>(tn, map, p, sms, stream);
}

}  // namespace lkv
