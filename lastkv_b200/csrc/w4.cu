// Products with 4-bit weights and group scales (sm_100a):
//   y[t, n] = sum_k x[t, k] * s[n, k / G] * c[n, k] (+ bias[n]),   c = -8 .. 7
// for x bf16, or int8 rows with fp32 group scales of the same G (rows_q8.cu).  Inside a
// group the products are summed unscaled - exactly, in int32, for int8 rows; in fp32 for
// bf16 rows, where c is exact in bf16 - and each group's sum is scaled once in fp32, so
// no weight is rounded after its 4 bits.
// w4.cuh has the packed layout; w4_tile.cu the kernel for more tokens.

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "ring.cuh"
#include "w4.cuh"

namespace lkv {

namespace {

// ---------------------------------------------------------------- packing

__global__ void __launch_bounds__(256)
    w4_pack_kernel(const uint8_t* __restrict__ codes, int64_t codes_row, const __nv_bfloat16* __restrict__ scales,
                   int64_t scales_row, int64_t n, int64_t k, int group, int kblocks, int row_blocks,
                   uint8_t* __restrict__ packed) {
  const int64_t rb = blockIdx.x / kblocks, kb = blockIdx.x % kblocks;
  const int64_t row0 = rb * kTileRows, k0 = kb * kTileK;
  uint8_t* dst = packed + block_offset(rb, kb, kblocks, row_blocks, group);
  for (int w = threadIdx.x; w < kCodeBytes / 4; w += blockDim.x) {
    const int i = w & 3, lane = (w >> 2) & 31, j = (w >> 7) & 1, r = w >> 8;
    const int64_t row = row0 + 16 * r + (lane >> 2) + 8 * (i & 1);
    const int64_t col = k0 + 32 * (2 * j + (i >> 1)) + 8 * (lane & 3);
    uint32_t word = 0;
    if (row < n && col < k) {
      const uint8_t* c = codes + row * codes_row + col / 2;  // bytes of column pairs (0,1) (2,3) (4,5) (6,7)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t lo = c[b >> 1] >> (4 * (b & 1)) & 15, hi = c[2 + (b >> 1)] >> (4 * (b & 1)) & 15;
        word |= ((lo ^ 8) | (hi ^ 8) << 4) << (8 * b);  // code u stands for u - 8
      }
    }
    reinterpret_cast<uint32_t*>(dst)[w] = word;
  }
  const int64_t groups = (k + group - 1) / group;
  for (int i = threadIdx.x; i < kTileRows * (kTileK / group); i += blockDim.x) {
    const int gi = i / kTileRows, e = i % kTileRows;
    const int64_t row = row0 + 16 * ((e >> 1) & 1) + 8 * (e & 1) + (e >> 2);
    const int64_t g = k0 / group + gi;
    const bool in = row < n && g < groups;
    reinterpret_cast<__nv_bfloat16*>(dst + kCodeBytes)[i] = in ? scales[row * scales_row + g] : __float2bfloat16(0.f);
  }
}

// Launched after w4_pack_kernel: the products read their weights before their launch's
// dependency wait (PDL), which a plain kernel in between makes safe - it starts once the
// packing has completed and its writes are visible, and the product's launch after it.
__global__ void w4_packed_kernel() {}

// ---------------------------------------------------------------- few tokens

struct SkinnyParams {
  const uint8_t* packed;
  const void* x;
  int64_t x_row;
  const float* x_scale;
  int64_t x_scale_row;
  const __nv_bfloat16* bias;
  __nv_bfloat16* y;
  int64_t y_row;
  int tokens, n, k, kblocks, splits, tiles;
  int* err;
  Never never;
};

__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A block's codes and scales in registers: 2 sub-tiles of 16 rows.
template <int G>
struct WeightBlock {
  uint4 w[2][2];
  uint2 s[kTileK / G];  // scales of rows g, g + 8 of each sub-tile
  __device__ __forceinline__ void read(const uint8_t* block, int lane) {  // from shared memory
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < 2; ++j) w[r][j] = ld_shared16(block + r * 1024 + j * 512 + lane * 16);
#pragma unroll
    for (int g = 0; g < kTileK / G; ++g)
      s[g] = ld_shared8(block + kCodeBytes + g * 64 + (lane >> 2) * 8);
  }
  // of every load's result
  __device__ __forceinline__ uint32_t mix() const {
    uint32_t v = w[0][0].x ^ w[0][1].x ^ w[1][0].x ^ w[1][1].x;
#pragma unroll
    for (int g = 0; g < kTileK / G; ++g) v ^= s[g].x;
    return v;
  }
  __device__ __forceinline__ uint32_t word(int r, int step, int half) const {
    const uint4& v = w[r][step >> 1];
    return (step & 1) ? (half ? v.w : v.z) : (half ? v.y : v.x);
  }
  __device__ __forceinline__ float scale(int g, int r, int half) const {
    const uint32_t v = r ? s[g].y : s[g].x;
    return half ? bf16_hi(v) : bf16_lo(v);
  }
};

// The rows' fragments of one group: int8 8 bytes, bf16 16 bytes per token and 32 columns.
template <bool INT8>
using XFrag = typename std::conditional<INT8, uint2, uint4>::type;

template <bool INT8>
__device__ __forceinline__ XFrag<INT8> x_load(const void* p) {
  return *reinterpret_cast<const XFrag<INT8>*>(p);
}

// One group of a block: acc += scaled products of its 32 rows and the tokens.
//   x:  fragments [NT][G / 32], rows as loaded;  xs: the tokens' scales (int8 rows)
template <bool INT8, int G, int NT>
__device__ __forceinline__ void add_group(float (&acc)[2][NT][4], const WeightBlock<G>& w, int gi,
                                          const XFrag<INT8> (&x)[NT][G / 32], const float (&xs)[NT][2]) {
  constexpr int kSteps = G / 32;
  if constexpr (INT8) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      // sums start at the bits of 1.5 * 2^23: read as fp32 they are 1.5 * 2^23 + sum (below 2^21), exactly
      int d[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[nt][e] = 0x4b400000;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t lo = w.word(r, gi * kSteps + s, 0), hi = w.word(r, gi * kSteps + s, 1);
        // codes in the upper half of each byte: 16 c
        const uint32_t a0 = lo * 16u & 0xf0f0f0f0u, a1 = hi * 16u & 0xf0f0f0f0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_s8_16832(d[nt], a0, a1, lo & 0xf0f0f0f0u, hi & 0xf0f0f0f0u, x[nt][s].x, x[nt][s].y);
      }
      const float s0 = w.scale(gi, r, 0) * 0.0625f, s1 = w.scale(gi, r, 1) * 0.0625f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[r][nt][e] = fmaf(__int_as_float(d[nt][e]) - 12582912.f, (e < 2 ? s0 : s1) * xs[nt][e & 1], acc[r][nt][e]);
    }
  } else {
    uint4 b[NT][kSteps];  // columns in the order of codes_bf16: (0, 2) (4, 6) (1, 3) (5, 7)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint4 v = x[nt][s];
        b[nt][s] = make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.z, v.w, 0x5410),
                              __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x7632));
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float d[NT][4] = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t lo = w.word(r, gi * kSteps + s, 0), hi = w.word(r, gi * kSteps + s, 1);
        const uint32_t a0 = codes_bf16<0>(lo), a1 = codes_bf16<0>(hi), a2 = codes_bf16<1>(lo), a3 = codes_bf16<1>(hi),
                       a4 = codes_bf16<2>(lo), a5 = codes_bf16<2>(hi), a6 = codes_bf16<3>(lo), a7 = codes_bf16<3>(hi);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_bf16_16816(d[nt], a0, a1, a2, a3, b[nt][s].x, b[nt][s].y);
          mma_bf16_16816(d[nt], a4, a5, a6, a7, b[nt][s].z, b[nt][s].w);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][nt][e] = fmaf(d[nt][e], w.scale(gi, r, e >> 1), acc[r][nt][e]);
    }
  }
}

// CTA = tiles of 32 output rows x 8 NT tokens, one split of k.  Its W warps take neighbouring
// runs of 128-column blocks; a warp streams its blocks through a ring of its own in shared
// memory by bulk copies (kDepth in flight, across the tiles' ends: kDepth x W x 2 KB per CTA
// cover the memory's latency).  The warps' sums meet in shared memory, the
// splits' sums (a cluster's CTAs, then one tile per CTA) over the cluster's, always in the
// same order.  Without splits the CTAs are persistent over the row tiles.  Tokens past the
// last read the last one's row (their sums are not stored).
// What it waits for, before HBM, with four warps a scheduler and half of the issue slots used:
// int8 rows for the activations and their scales, loaded in the iteration that uses them (the
// largest stall), bf16 rows for their 1.4 times as many instructions, most of them the expansion;
// small weights for the launch and the memory's latency.  8 tokens, groups of 128, int8 / bf16
// rows: 28672 x 4096 13.9 / 19.3 us (4.4 / 3.2 TB/s of the 6.5 measured), 4096 x 14336 7.8 / 10.3
// us, 4096 x 4096 3.6 / 4.4 us; 1 token, 6144 x 4096 4.0 / 6.0 us.  Three CTAs per SM (85 registers) were no faster,
// the round that 896 tiles begin on 296 CTAs costs 0.9 / 1.6 us.
// Loads into registers instead of the ring: 15.9 / 23.3 us for the first.
// kDepth: three blocks of 16 warps are 101 KB in flight per SM, above what the latency asks for
// (6.5 TB/s x 1 us / 148 SMs = 44 KB).
constexpr int kDepth = 3;
constexpr int kSkinnyKernelId = 14;

template <int G, int NT, int W>
struct SkinnyShared {
  alignas(128) uint8_t ring[W][kDepth][block_bytes(G)];
  float red[2][W][8 * NT][kTileRows + 4];  // 4: the fragments' stores stay off each other's banks
  float part[8 * NT][kTileRows];
  uint64_t full[W][kDepth];
};

template <bool INT8, int G, int NT, int W>
__global__ void __launch_bounds__(W * 32, 16 / W) w4_skinny_kernel(const SkinnyParams p) {
  extern __shared__ uint8_t smem_raw[];
  using Sh = SkinnyShared<G, NT, W>;
  Sh* sh = reinterpret_cast<Sh*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  constexpr int kTok = 8 * NT, kSteps = G / 32, kElem = INT8 ? 1 : 2, kRows = kTileRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.y, tok0 = blockIdx.z * kTok;
  const int c0 = (int)((int64_t)p.kblocks * split / p.splits), c1 = (int)((int64_t)p.kblocks * (split + 1) / p.splits);
  const int k0 = c0 + (c1 - c0) * warp / W, k1 = c0 + (c1 - c0) * (warp + 1) / W;
  const int whole = p.k / kTileK;  // blocks below are whole
  pdl_launch_dependents();
  if (lane == 0) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) mbar_init(&sh->full[warp][d], 1);
    fence_barrier_init();
  }
  __syncwarp();
  // load cursor: a tile's blocks [k0, k1), then the CTA's next tile
  int lt = k0 < k1 ? (int)blockIdx.x : p.tiles, lk = k0;
  Ring<kDepth> ring;
  auto load = [&] {
    if (lt >= p.tiles) return;
    const int slot = ring.fill();
    if (lane == 0) {
      mbar_arrive_expect_tx(&sh->full[warp][slot], block_bytes(G));
      bulk_load_hint(sh->ring[warp][slot], p.packed + block_offset(lt, lk, p.kblocks, p.tiles, G), block_bytes(G),
                     &sh->full[warp][slot], policy_evict_first());
    }
    if (++lk == k1) {
      lk = k0;
      lt += gridDim.x;
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) load();  // the weights do not depend on the previous kernel
  const uint8_t* xp[NT];
  const float* sp[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int64_t tok = min(tok0 + 8 * nt + g, p.tokens - 1);
    xp[nt] = static_cast<const uint8_t*>(p.x) + (tok * p.x_row + 8 * t) * kElem;
#pragma unroll
    for (int h = 0; h < 2; ++h) sp[nt][h] = p.x_scale + min(tok0 + 8 * nt + 2 * t + h, p.tokens - 1) * p.x_scale_row;
  }
  pdl_wait();

  bool ok = true;
  for (int tile = blockIdx.x, buf = 0; tile < p.tiles; tile += gridDim.x, buf ^= 1) {
    float acc[2][NT][4] = {};
    for (int kb = k0; ok && kb < k1; ++kb) {
      const int64_t at = (int64_t)kb * kTileK * kElem;
      XFrag<INT8> x[NT][4];
      float xs[NT][kTileK / G][2];
      if (kb < whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int s = 0; s < 4; ++s) x[nt][s] = x_load<INT8>(xp[nt] + at + 32 * s * kElem);
#pragma unroll
          for (int gi = 0; gi < kTileK / G; ++gi)
#pragma unroll
            for (int h = 0; h < 2; ++h) xs[nt][gi][h] = INT8 ? sp[nt][h][kb * (kTileK / G) + gi] : 1.f;
        }
      } else {  // the block that the row ends in
        const int left = p.k - kb * kTileK;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int s = 0; s < 4; ++s)
            x[nt][s] = 32 * s + 8 * t < left ? x_load<INT8>(xp[nt] + at + 32 * s * kElem) : XFrag<INT8>{};
#pragma unroll
          for (int gi = 0; gi < kTileK / G; ++gi)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              xs[nt][gi][h] = INT8 && gi * G < left ? sp[nt][h][kb * (kTileK / G) + gi] : 0.f;
        }
      }
      ok = mbar_wait(&sh->full[warp][ring.slot], ring.phase);
      WeightBlock<G> w;
      w.read(sh->ring[warp][ring.slot], lane);
      // every lane's block is in registers: its slot may be filled again
      ok = !__any_sync(0xffffffffu, !ok || p.never.is(w.mix()));
      if (!ok) break;  // this block's copy, and those behind it, are still in flight
      ring.next();
      load();
#pragma unroll
      for (int gi = 0; gi < kTileK / G; ++gi) {
        XFrag<INT8> xg[NT][kSteps];
        float sg[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int s = 0; s < kSteps; ++s) xg[nt][s] = x[nt][gi * kSteps + s];
          sg[nt][0] = xs[nt][gi][0], sg[nt][1] = xs[nt][gi][1];
        }
        add_group<INT8, G, NT>(acc, w, gi, xg, sg);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sh->red[buf][warp][8 * nt + 2 * t + (e & 1)][16 * r + g + 8 * (e >> 1)] = acc[r][nt][e];
    __syncthreads();  // one barrier per tile: the next one's sums go to the other buffer
    const int live = min(kTok, p.tokens - tok0) * kRows;
    for (int i = threadIdx.x; i < live; i += W * 32) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += sh->red[buf][w][i / kRows][i % kRows];
      if (p.splits > 1) {
        sh->part[i / kRows][i % kRows] = sum;
      } else {
        const int row = tile * kRows + i % kRows;
        if (row < p.n) {
          if (p.bias) sum += __bfloat162float(p.bias[row]);
          p.y[(int64_t)(tok0 + i / kRows) * p.y_row + row] = __float2bfloat16_rn(sum);
        }
      }
    }
  }
  if (!ok) {
    if (lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, kSkinnyKernelId, warp);
    // no copy may still be in flight when the CTA leaves
    for (; ring.flying > 0; ring.next()) mbar_wait(&sh->full[warp][ring.slot], ring.phase);
  }
  if (p.splits > 1) {
    const int tile = blockIdx.x;
    const int live = min(kTok, p.tokens - tok0) * kRows;
    cluster_sync_all();  // every split has published its sums
    const uint32_t base = smem_u32(&sh->part[0][0]);
    const int rank = (int)cluster_rank();
    for (int i = rank * (W * 32) + threadIdx.x; i < live; i += p.splits * W * 32) {
      float sum = 0.f;
      for (int s = 0; s < p.splits; ++s) sum += dsmem_ld(dsmem_map(base, s) + i * 4);
      const int row = tile * kRows + i % kRows;
      if (row < p.n) {
        if (p.bias) sum += __bfloat162float(p.bias[row]);
        p.y[(int64_t)(tok0 + i / kRows) * p.y_row + row] = __float2bfloat16_rn(sum);
      }
    }
    cluster_sync_all();  // the sums stay readable until every CTA has read them
  }
}

// Splits of k over a cluster (a power of two <= 8): while every CTA still has an SM and a
// warp about two blocks.  8 tokens, 1024 x 14336, int8 / bf16 rows: 5.96 / 8.71 us without,
// 4.68 / 5.47 us with four; 1024 x 8192 with one block per warp (four) 3.79 / 4.23 us, with
// two 3.82 / 4.46 us; 256 x 4096 2.69 / 3.36 us without, 3.09 / 3.32 us with two.
int choose_splits(int64_t ctas, int kblocks, int sms, int warps) {
  int s = 1;
  while (s < 8 && ctas * s * 2 <= sms && kblocks >= 3 * s * warps) s *= 2;
  return s;
}

template <bool INT8, int G, int NT, int W>
int launch_skinny(SkinnyParams p, int sms, cudaStream_t stream) {
  constexpr int kSmem = sizeof(SkinnyShared<G, NT, W>) + 128;
  auto kernel = w4_skinny_kernel<INT8, G, NT, W>;
  static std::once_flag once[64];
  static cudaError_t set[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LKV_ERR_CUDA;
  std::call_once(once[dev], [&] {
    set[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (set[dev] != cudaSuccess) return LKV_ERR_CUDA;
  const int64_t slots = 16 / W * sms, ztiles = (p.tokens + 8 * NT - 1) / (8 * NT);
  p.splits = choose_splits(p.tiles * ztiles, p.kblocks, sms, W);
  const int ctas = p.splits > 1 ? p.tiles : (int)std::min<int64_t>(p.tiles, std::max<int64_t>(1, slots / ztiles));
  return launch_pdl_cluster(kernel, dim3(ctas, p.splits, (unsigned)ztiles), dim3(W * 32), kSmem, stream,
                            dim3(1, p.splits, 1), p) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

// 16 warps per row tile while every tile has an SM to itself, else two CTAs of 8 per SM.
// 8 tokens, int8 / bf16 rows, 16 against 8 warps: 4096 x 4096 (128 tiles) 3.70 / 4.45 against
// 4.13 / 5.73 us, 4096 x 14336 7.95 / 10.3 against 11.4 / 16.9 us; 6144 x 4096 (192 tiles)
// 5.25 / 6.22 against 4.72 / 5.96 us, 28672 x 4096 15.5 / 20.0 against 13.9 / 19.3 us.
template <bool INT8, int G>
int skinny(const SkinnyParams& p, int sms, cudaStream_t stream) {
  const bool wide = (int64_t)p.tiles * ((p.tokens + 15) / 16) <= sms;
  if (p.tokens <= 8)
    return wide ? launch_skinny<INT8, G, 1, 16>(p, sms, stream) : launch_skinny<INT8, G, 1, 8>(p, sms, stream);
  return wide ? launch_skinny<INT8, G, 2, 16>(p, sms, stream) : launch_skinny<INT8, G, 2, 8>(p, sms, stream);
}

int device_sms(int* sms) {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LKV_ERR_CUDA;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return LKV_ERR_CUDA;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return LKV_OK;
}

// The streaming kernel reads the weight again for every 16 tokens (from L2), so it takes up to
// 32 tokens, and more where its CTAs still fit the GPU at once; the tcgen05 kernel the rest.
// int8 / bf16 rows, streaming against tcgen05: 32 tokens 4096 x 4096 6.1 / 7.8 against 9.5 /
// 11.6 us, 28672 x 4096 34.7 / 48.7 against 36.9 / 53.0 us; 64 tokens 1003 x 1544 2.7 / 3.3
// against 5.9 / 6.9 us, 4096 x 4096 (512 CTAs) 10.9 / 14.3 against 9.9 / 12.0 us.
bool few_tokens(const W4Args& a, int sms) {
  return a.tokens <= 32 || (a.n + kTileRows - 1) / kTileRows * ((a.tokens + 15) / 16) <= 2 * (int64_t)sms;
}

constexpr int64_t kMaxTokens = 16 * 65535;  // the streaming kernel's grid

bool shape_ok(int64_t n, int64_t k) { return n >= 1 && n <= 0x7fffff00 && k >= 8 && k <= 0x7fffff00 && k % 8 == 0; }

}  // namespace

size_t w4_bytes(int64_t n, int64_t k, int group) {
  if ((group != 32 && group != 64 && group != 128) || !shape_ok(n, k)) return 0;
  return (size_t)((n + kTileRows - 1) / kTileRows) * (size_t)((k + kTileK - 1) / kTileK) * block_bytes(group);
}

int w4_pack(const uint8_t* codes, int64_t codes_row, const void* scales, int64_t scales_row, int64_t n, int64_t k,
            int group, void* packed, cudaStream_t stream) {
  if (group != 32 && group != 64 && group != 128) return LKV_ERR_UNSUPPORTED;
  if (!shape_ok(n, k) || !codes || !scales || !packed || (reinterpret_cast<uintptr_t>(packed) & 15) ||
      (reinterpret_cast<uintptr_t>(scales) & 1) ||
      (n > 1 && (codes_row < k / 2 || scales_row < (k + group - 1) / group)))
    return LKV_ERR_INVALID_ARGUMENT;
  const int64_t kblocks = (k + kTileK - 1) / kTileK, blocks = (n + kTileRows - 1) / kTileRows * kblocks;
  if (blocks > 0x7fffffff) return LKV_ERR_UNSUPPORTED;
  w4_pack_kernel<<<(unsigned)blocks, 256, 0, stream>>>(codes, codes_row, static_cast<const __nv_bfloat16*>(scales),
                                                       scales_row, n, k, group, (int)kblocks, (int)(blocks / kblocks),
                                                       static_cast<uint8_t*>(packed));
  w4_packed_kernel<<<1, 1, 0, stream>>>();
  return cudaGetLastError() == cudaSuccess ? LKV_OK : LKV_ERR_CUDA;
}

int w4_linear(const W4Args& a, cudaStream_t stream) {
  if (a.group != 32 && a.group != 64 && a.group != 128) return LKV_ERR_UNSUPPORTED;
  if (!shape_ok(a.n, a.k) || a.tokens < 0 || a.tokens > kMaxTokens) return LKV_ERR_INVALID_ARGUMENT;
  if (a.tokens == 0) return LKV_OK;
  const bool int8 = a.x_scale != nullptr;
  const int align = int8 ? 8 : 16, elem = int8 ? 1 : 2;
  if (!a.x || !a.packed || !a.y || (reinterpret_cast<uintptr_t>(a.packed) & 15) ||
      (reinterpret_cast<uintptr_t>(a.x) % align) || (reinterpret_cast<uintptr_t>(a.y) & 1) ||
      (reinterpret_cast<uintptr_t>(a.bias) & 1) || (reinterpret_cast<uintptr_t>(a.x_scale) & 3))
    return LKV_ERR_INVALID_ARGUMENT;
  if (a.tokens > 1 && ((a.x_row * elem) % align || a.x_row < a.k || a.y_row < a.n ||
                       (int8 && a.x_scale_row < (a.k + a.group - 1) / a.group)))
    return LKV_ERR_INVALID_ARGUMENT;
  int sms = 0;
  const int st = device_sms(&sms);
  if (st != LKV_OK) return st;
  if (!few_tokens(a, sms) && w4_tile_aligned(a)) return w4_tile(a, sms, stream);
  SkinnyParams p{};
  p.packed = static_cast<const uint8_t*>(a.packed);
  p.x = a.x;
  p.x_row = a.x_row;
  p.x_scale = a.x_scale;
  p.x_scale_row = a.x_scale_row;
  p.bias = static_cast<const __nv_bfloat16*>(a.bias);
  p.y = static_cast<__nv_bfloat16*>(a.y);
  p.y_row = a.y_row;
  p.tokens = (int)a.tokens;
  p.n = (int)a.n;
  p.k = (int)a.k;
  p.kblocks = (int)((a.k + kTileK - 1) / kTileK);
  p.tiles = (int)((a.n + kTileRows - 1) / kTileRows);
  p.err = a.error_word;
  if (int8)
    return a.group == 32   ? skinny<true, 32>(p, sms, stream)
           : a.group == 64 ? skinny<true, 64>(p, sms, stream)
                           : skinny<true, 128>(p, sms, stream);
  return a.group == 32   ? skinny<false, 32>(p, sms, stream)
         : a.group == 64 ? skinny<false, 64>(p, sms, stream)
                         : skinny<false, 128>(p, sms, stream);
}

}  // namespace lkv
