// Products with 4-bit weights for many bf16 rows, on tcgen05 (sm_100a).
//
// Tile: 128 output rows (the MMA's M side) x TN tokens (N side), summed over all of k in
// TMEM.  Per 64 columns one stage of shared memory holds the A operand - the weights
// bf16(s * c), expanded from their 4 bits by eight warps - and the B operand, the rows as
// they are, by TMA; both K-major, 128-byte swizzled.
//
// The scales go into the operand because sums that leave TMEM after every group cost the
// tensor core as much as they take to read: with group sums scaled in fp32 on their way out
// (as w4_tile.cu does for int8 rows, whose operands have no room for a scale) 2048 tokens x
// 28672 x 4096 took 455 us.  The price is one rounding of s * c, which has up to 12
// significant bits, to 8; like the rounding of the output it is 2^-9 of the weight at most and
// unrelated from weight to weight.
//
// Roles of the 512 threads (one CTA per SM, persistent over the tiles):
//   warp 0  rows by TMA    warp 1  tcgen05.mma issue, TMEM    warp 3  weights by bulk copies
//   warps 4-11  weights -> A tiles, the two warpgroups a stage each in turn
//   warps 12-15 epilogue of a tile while the next one is summed in the other TMEM buffer
// Where the tiles alone do not fill the GPU, k is split over the CTAs of a cluster, whose
// partial tiles meet in shared memory (added in split order).

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "tcgen05.cuh"
#include "w4.cuh"

namespace lkv {

namespace {

constexpr int kM = 128;
constexpr int kQuarters = kM / kTileRows;  // packed row blocks of a tile
constexpr int kThreads = 512;
constexpr int kKernelId = 15;
constexpr int kAStage = kM * 128;
constexpr int kMaxSplits = 8;

struct WideParams {
  const uint8_t* packed;
  const __nv_bfloat16* bias;
  __nv_bfloat16* y;
  int64_t y_row;
  int tokens, n, kblocks, row_blocks, tok_tiles, tiles, splits;
  int* err;
};

// Ring depths: A stages (16 KB, filled in the CTA), B stages (TN x 128 bytes, from L2), and
// 128-column blocks of packed weights (8 KB and the scales for the tile's 128 rows).
template <int TN>
__host__ __device__ constexpr int a_stages() {
  return TN == 256 ? 4 : 6;
}
template <int TN>
__host__ __device__ constexpr int b_stages() {
  return TN == 256 ? 4 : TN == 128 ? 6 : 8;
}
template <int TN>
__host__ __device__ constexpr int code_slots() {
  return TN == 64 ? 6 : 3;
}

template <int G, int TN>
__host__ __device__ constexpr int ring_bytes() {
  return a_stages<TN>() * kAStage + b_stages<TN>() * TN * 128 + code_slots<TN>() * kQuarters * block_bytes(G);
}

template <int TN>
struct Shared {
  uint64_t a_full[a_stages<TN>()], a_empty[a_stages<TN>()];
  uint64_t b_full[b_stages<TN>()], b_empty[b_stages<TN>()];
  uint64_t c_full[code_slots<TN>()], c_empty[code_slots<TN>()];
  uint64_t d_full[2], d_empty[2];
  uint64_t done;
  uint32_t tmem;
};

template <int G, int TN>
constexpr int smem_bytes() {
  return 1024 + ring_bytes<G, TN>() + (int)sizeof(Shared<TN>);
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 v =
      __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int G, int TN>
__global__ void __launch_bounds__(kThreads, 1)
    w4_wide_kernel(const __grid_constant__ CUtensorMap tmx, const WideParams p) {
  constexpr int SA = a_stages<TN>(), SB = b_stages<TN>(), C = code_slots<TN>(), kBStage = TN * 128;
  constexpr uint32_t kIdesc = umma_idesc_bf16(kM, TN, 0, 0);
  constexpr uint32_t kTmemCols = 2 * TN;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* b_ring = smem + SA * kAStage;
  uint8_t* codes = b_ring + SB * kBStage;  // [C][kQuarters][block_bytes(G)]
  Shared<TN>* sh = reinterpret_cast<Shared<TN>*>(smem + ring_bytes<G, TN>());
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
    for (int b = 0; b < C; ++b) {
      mbar_init(&sh->c_full[b], 1);
      mbar_init(&sh->c_empty[b], 8);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sh->d_full[b], 1);
      mbar_init(&sh->d_empty[b], 4);
    }
    mbar_init(&sh->done, 1);
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

  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------------- rows by TMA
      tma_prefetch_desc(&tmx);
      pdl_wait();
      uint32_t it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
        const int tok0 = tile % p.tok_tiles * TN;
        for (int i = 0; i < nkb * 2; ++i, ++it) {
          const int s = it % SB;
          ok = mbar_wait(&sh->b_empty[s], ((it / SB) & 1) ^ 1);
          if (!ok) break;
          mbar_arrive_expect_tx(&sh->b_full[s], kBStage);
          tma_load_2d(b_ring + s * kBStage, &tmx, &sh->b_full[s], (kb0 * 2 + i) * 64, tok0);
        }
      }
      if (!ok) {  // no copy may still be in flight when the CTA leaves
        report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, (int)it);
        for (uint32_t i = it > SB ? it - SB : 0; i < it; ++i) mbar_wait(&sh->b_full[i % SB], (i / SB) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    const uint64_t desc_a = umma_sdesc_sw128(smem_u32(smem), 16, 1024);
    const uint64_t desc_b = umma_sdesc_sw128(smem_u32(b_ring), 16, 1024);
    uint32_t sa = 0, sb = 0, pa = 0, pb = 0, buf = 0, pd = 1, it = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      ok = mbar_wait(&sh->d_empty[buf], pd);
      for (int i = 0; i < nkb * 2; ++i, ++it) {
        ok = ok && mbar_wait(&sh->a_full[sa], pa) && mbar_wait(&sh->b_full[sb], pb);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t da = desc_a + sa * (kAStage >> 4), db = desc_b + sb * (kBStage >> 4);
#pragma unroll
          for (int m = 0; m < 4; ++m)  // 32 bytes of k each: 2 in descriptor units
            umma_bf16_ss(tmem + buf * TN, da + 2 * m, db + 2 * m, kIdesc, i > 0 || m > 0);
          umma_commit(&sh->a_empty[sa]);
          umma_commit(&sh->b_empty[sb]);
          if (i == nkb * 2 - 1) umma_commit(&sh->d_full[buf]);
        }
        __syncwarp();
        if (++sa == SA) sa = 0, pa ^= 1;
        if (++sb == SB) sb = 0, pb ^= 1;
      }
      buf ^= 1;
      if (buf == 0) pd ^= 1;
    }
    if (!ok && lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 1000000 + (int)it);
    if (elect_one()) umma_commit(&sh->done);
    __syncwarp();
    mbar_wait(&sh->done, 0);  // no MMA may still be in flight when TMEM is freed
  } else if (warp == 3) {
    // ------------------------------------------------------------------ packed weights by bulk copies
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
      if (!ok) {
        report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 5000000 + (int)blk);
        for (uint32_t i = blk > C ? blk - C : 0; i < blk; ++i) mbar_wait(&sh->c_full[i % C], (i / C) & 1);
      }
    }
  } else if (warp >= 4 && warp < 12) {
    // ------------------------------------------------------------------ weights -> A tiles
    // Warp w of a warpgroup expands row block w, the warpgroup `own` the block's 64 columns
    // from 64 own on.  Piece of lane 4 g + t: a phase of eight lanes reads all eight 16-byte
    // banks of its 128 bytes (t and the parity of g) and stores to all eight swizzled chunks
    // (chunk ^ g), the rows of a phase being g and g ^ 5.
    const int w = warp & 3, own = (warp >> 2) - 1, t = lane & 3, q3 = lane >> 3;
    const int g = ((q3 & 1) << 1 | q3 >> 1) ^ ((lane & 4) ? 5 : 0);
    uint32_t blk = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      const int quarters = min(kQuarters, p.row_blocks - tile / p.tok_tiles * kQuarters);
      for (int kb = 0; kb < nkb; ++kb, ++blk) {
        const int b = blk % C;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->c_full[b], (blk / C) & 1));
        if (!ok) break;
        const uint8_t* src = codes + (b * kQuarters + w) * block_bytes(G);
        uint4 v[2];
        uint2 scales[2];  // of the two 32-column steps: rows g, g + 8 of both sub-tiles
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          v[r] = w < quarters ? *reinterpret_cast<const uint4*>(src + r * 1024 + own * 512 + (4 * g + t) * 16)
                              : make_uint4(0, 0, 0, 0);
          scales[r] = w < quarters ? *reinterpret_cast<const uint2*>(src + kCodeBytes + (64 * own + 32 * r) / G * 64 + g * 8)
                                   : make_uint2(0, 0);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->c_empty[b]);
        const uint32_t it = blk * 2 + own;
        const int s = it % SA;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh->a_empty[s], ((it / SA) & 1) ^ 1));
        if (!ok) break;
        const uint32_t a = smem_u32(smem + s * kAStage);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t words[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // row 16 r + 8 (e & 1) + g, step e / 2
            const uint32_t u = words[e], pair = r ? scales[e >> 1].y : scales[e >> 1].x;
            const uint32_t sc = __byte_perm(pair, pair, (e & 1) ? 0x3232 : 0x1010);
            const uint32_t c02 = mul_bf16x2(codes_bf16<0>(u), sc), c46 = mul_bf16x2(codes_bf16<1>(u), sc),
                           c13 = mul_bf16x2(codes_bf16<2>(u), sc), c57 = mul_bf16x2(codes_bf16<3>(u), sc);
            const uint32_t row = a + (w * kTileRows + 16 * r + 8 * (e & 1) + g) * 128;
            const int chunk = 4 * (e >> 1) + t;
            st_shared16(row + ((chunk ^ g) << 4), __byte_perm(c02, c13, 0x5410), __byte_perm(c02, c13, 0x7632),
                        __byte_perm(c46, c57, 0x5410), __byte_perm(c46, c57, 0x7632));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->a_full[s]);
      }
    }
    if (!ok && lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 2000000 + (int)blk);
  } else if (warp >= 12) {
    // ------------------------------------------------------------------ epilogue
    const int sub = warp & 3, g = lane >> 2, q = lane & 3;
    const uint32_t lanes = (uint32_t)(sub * 32) << 16;
    const bool words = ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)(p.y_row * 2)) & 3) == 0;
    uint32_t buf = 0, phase = 0;
    bool ok = true;
    pdl_wait();  // before any global write
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
      const int tok0 = tile % p.tok_tiles * TN, row0 = (tile / p.tok_tiles) * kM + sub * kTileRows;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh->d_full[buf], phase));
      if (!ok) break;
      tc_fence_after();
      const uint32_t at = tmem + lanes + buf * TN;
      float bias[2][2] = {};
      if (p.bias && p.splits == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = row0 + 16 * h + 8 * e + g;
            if (r < p.n) bias[h][e] = __bfloat162float(p.bias[r]);
          }
      }
      // one tile per cluster: every stage has been consumed, their memory takes the partial [token][row]
      float* part = reinterpret_cast<float*>(smem) + 2 * q * kM + sub * kTileRows + g;
#pragma unroll 1
      for (int c0 = 0; c0 < TN; c0 += 16) {
        uint32_t u[2][8];
        tmem_ld_16x16(at + c0, u[0]);
        tmem_ld_16x16(at + (16u << 16) + c0, u[1]);
        tmem_wait_ld16(u);
        if (c0 + 16 == TN) {  // the buffer is read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->d_empty[buf]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float lo = __uint_as_float(u[h][4 * c + 2 * e]), hi = __uint_as_float(u[h][4 * c + 2 * e + 1]);
              if (p.splits > 1) {
                part[(c0 + 8 * c) * kM + 16 * h + 8 * e] = lo;
                part[(c0 + 8 * c + 1) * kM + 16 * h + 8 * e] = hi;
                continue;
              }
              // 8 rows x 8 tokens through a register transpose: a lane then stores two
              // neighbouring rows of one token
              const uint32_t v = movmatrix_trans(pack_bf16(lo + bias[h][e], hi + bias[h][e]));
              const int tok = tok0 + c0 + 8 * c + g, f = row0 + 16 * h + 8 * e + 2 * q;
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
      buf ^= 1;
      if (buf == 0) phase ^= 1;
    }
    if (!ok && lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kKernelId, 3000000);
  }

  __syncwarp();
  if (p.splits > 1) {
    cluster_sync_all();  // every split has published its partial
    const int tile = blockIdx.x;
    const int tok0 = tile % p.tok_tiles * TN, row0 = tile / p.tok_tiles * kM;
    const int live = min(TN, p.tokens - tok0) * kM;
    const uint32_t base = smem_u32(smem);
    for (int i = (int)cluster_rank() * kThreads + threadIdx.x; i < live; i += p.splits * kThreads) {
      const int r = row0 + i % kM;
      float v[kMaxSplits];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) v[s] = s < p.splits ? dsmem_ld(dsmem_map(base, s) + i * 4) : 0.f;
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) sum += v[s];
      if (r < p.n) {
        if (p.bias) sum += __bfloat162float(p.bias[r]);
        p.y[(int64_t)(tok0 + i / kM) * p.y_row + r] = __float2bfloat16_rn(sum);
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

template <int G, int TN>
int launch(const CUtensorMap& map, const WideParams& p, int sms, cudaStream_t stream) {
  static_assert(smem_bytes<G, TN>() <= 227 * 1024, "shared memory of a CTA");
  static std::once_flag once[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LKV_ERR_CUDA;
  static cudaError_t set[64];
  std::call_once(once[dev], [&] {
    set[dev] = cudaFuncSetAttribute(w4_wide_kernel<G, TN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    smem_bytes<G, TN>());
  });
  if (set[dev] != cudaSuccess) return LKV_ERR_CUDA;
  const dim3 grid(std::min(p.tiles, std::max(1, sms / p.splits)), p.splits);
  return launch_pdl_cluster(w4_wide_kernel<G, TN>, grid, dim3(kThreads), smem_bytes<G, TN>(), stream,
                            dim3(1, p.splits, 1), map, p) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

template <int G>
int by_tokens(int tn, const CUtensorMap& map, const WideParams& p, int sms, cudaStream_t stream) {
  return tn == 64    ? launch<G, 64>(map, p, sms, stream)
         : tn == 128 ? launch<G, 128>(map, p, sms, stream)
                     : launch<G, 256>(map, p, sms, stream);
}

}  // namespace

int w4_wide(const W4Args& a, int sms, cudaStream_t stream) {
  WideParams p{};
  p.packed = static_cast<const uint8_t*>(a.packed);
  p.bias = static_cast<const __nv_bfloat16*>(a.bias);
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.y_row = a.y_row;
  p.tokens = (int)a.tokens;
  p.n = (int)a.n;
  p.kblocks = (int)((a.k + kTileK - 1) / kTileK);
  p.row_blocks = (int)((a.n + kTileRows - 1) / kTileRows);
  p.err = a.error_word;
  const int tn = a.tokens <= 64 ? 64 : a.tokens <= 128 ? 128 : 256;
  p.tok_tiles = (int)((a.tokens + tn - 1) / tn);
  const int64_t tiles = (a.n + kM - 1) / kM * p.tok_tiles;
  if (tiles > 0x7fffffff) return LKV_ERR_UNSUPPORTED;
  p.tiles = (int)tiles;
  // a power of two of splits, while every CTA of every cluster still has an SM and two blocks of k
  p.splits = 1;
  while (p.splits < kMaxSplits && p.tiles * p.splits * 2 <= sms && p.kblocks >= p.splits * 4) p.splits *= 2;
  CUtensorMap map;
  const int st = make_matrix_tensor_map(&map, a.x, a.tokens, a.k, a.x_row, tn);
  if (st != LKV_OK) return st;
  return a.group == 32   ? by_tokens<32>(tn, map, p, sms, stream)
         : a.group == 64 ? by_tokens<64>(tn, map, p, sms, stream)
                         : by_tokens<128>(tn, map, p, sms, stream);
}

}  // namespace lkv
