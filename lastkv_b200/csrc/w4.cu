// Products with 4-bit weights and group scales (sm_100a):
//   y[t, n] = sum_k x[t, k] * s[n, k / G] * c[n, k] (+ bias[n]),   c = -8 .. 7
// for x bf16, or int8 rows with fp32 group scales of the same G (rows_q8.cu).  Inside a
// group the products are summed unscaled - exactly, in int32, for int8 rows; in fp32 for
// bf16 rows, where c is exact in bf16 - and each group's sum is scaled once in fp32, so
// no weight is rounded after its 4 bits.
// w4.cuh has the packed layout; w4_tile.cu the kernel for more tokens.

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "w4.cuh"

namespace lkv {

namespace {

// ---------------------------------------------------------------- packing

__global__ void __launch_bounds__(256)
    w4_pack_kernel(const uint8_t* __restrict__ codes, int64_t codes_row, const __nv_bfloat16* __restrict__ scales,
                   int64_t scales_row, int64_t n, int64_t k, int group, int64_t kblocks, uint8_t* __restrict__ packed) {
  const int64_t block = blockIdx.x;  // (row tile, k block)
  const int64_t row0 = block / kblocks * kTileRows, k0 = block % kblocks * kTileK;
  uint8_t* dst = packed + block * block_bytes(group);
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
    const int64_t row = row0 + 16 * ((e >> 1) & 3) + 8 * (e & 1) + (e >> 3);
    const int64_t g = k0 / group + gi;
    const bool in = row < n && g < groups;
    reinterpret_cast<__nv_bfloat16*>(dst + kCodeBytes)[i] = in ? scales[row * scales_row + g] : __float2bfloat16(0.f);
  }
}

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
  int tokens, n, k, kblocks, splits;
};

__device__ __forceinline__ void mma_s8_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

constexpr int kWarps = 8;
constexpr int kSkinnyTokens = 16;  // above, the tcgen05 kernel takes over
constexpr int kRedStride = kTileRows + 4;  // [token][row] partials; 4 keeps the fragment stores off each other's banks

template <int G>
struct WeightBlock {
  uint4 w[4][2];
  uint4 s[kTileK / G];
  __device__ __forceinline__ void load(const uint8_t* block, int lane) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      w[r][0] = ld_stream(block + r * 1024 + lane * 16);
      w[r][1] = ld_stream(block + r * 1024 + 512 + lane * 16);
    }
#pragma unroll
    for (int g = 0; g < kTileK / G; ++g) s[g] = ld_stream(block + kCodeBytes + g * 128 + (lane >> 2) * 16);
  }
  __device__ __forceinline__ uint32_t word(int r, int step, int half) const {
    const uint4& v = w[r][step >> 1];
    return (step & 1) ? (half ? v.w : v.z) : (half ? v.y : v.x);
  }
  __device__ __forceinline__ float scale(int g, int r, int half) const {
    const uint32_t v = r == 0 ? s[g].x : r == 1 ? s[g].y : r == 2 ? s[g].z : s[g].w;
    return half ? bf16_hi(v) : bf16_lo(v);
  }
};

// CTA = 64 output rows x 8 NT tokens x one split of k; its 8 warps take neighbouring
// runs of 128-column blocks and their sums meet in shared memory, the splits' sums over
// the cluster's shared memory, always in the same order.
template <bool INT8, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32) w4_skinny_kernel(const SkinnyParams p) {
  extern __shared__ float red[];  // [kWarps][8 NT][kRedStride], then the CTA's sums [8 NT][kTileRows]
  constexpr int kTok = 8 * NT, kSteps = G / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.x, split = blockIdx.y, tok0 = blockIdx.z * kTok;
  const int c0 = (int)((int64_t)p.kblocks * split / p.splits), c1 = (int)((int64_t)p.kblocks * (split + 1) / p.splits);
  const int k0 = c0 + (c1 - c0) * warp / kWarps, k1 = c0 + (c1 - c0) * (warp + 1) / kWarps;
  const uint8_t* wp = p.packed + ((int64_t)tile * p.kblocks + k0) * block_bytes(G);
  pdl_launch_dependents();
  WeightBlock<G> next;
  if (k0 < k1) next.load(wp, lane);  // the weights do not depend on the previous kernel
  pdl_wait();

  float acc[4][NT][4] = {};
  for (int kb = k0; kb < k1; ++kb) {
    const WeightBlock<G> cur = next;
    wp += block_bytes(G);
    if (kb + 1 < k1) next.load(wp, lane);
#pragma unroll
    for (int gi = 0; gi < kTileK / G; ++gi) {
      const int col = kb * kTileK + gi * G + 8 * t;
      if constexpr (INT8) {
        uint2 b[NT][kSteps];
        float xs[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int64_t tok = tok0 + 8 * nt + g;
          const int8_t* x = static_cast<const int8_t*>(p.x) + tok * p.x_row + col;
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
            b[nt][s] = tok < p.tokens && col + 32 * s < p.k ? *reinterpret_cast<const uint2*>(x + 32 * s)
                                                            : make_uint2(0, 0);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t dt = tok0 + 8 * nt + 2 * t + h;
            const int grp = kb * (kTileK / G) + gi;
            xs[nt][h] = dt < p.tokens && grp * G < p.k ? p.x_scale[dt * p.x_scale_row + grp] * 0.0625f : 0.f;
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          int d[NT][4] = {};
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const uint32_t lo = cur.word(r, gi * kSteps + s, 0), hi = cur.word(r, gi * kSteps + s, 1);
            // codes in the upper half of each byte: 16 c
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_s8_16832(d[nt], lo << 4 & 0xf0f0f0f0u, hi << 4 & 0xf0f0f0f0u, lo & 0xf0f0f0f0u, hi & 0xf0f0f0f0u,
                           b[nt][s].x, b[nt][s].y);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[r][nt][e] = fmaf((float)d[nt][e], cur.scale(gi, r, e >> 1) * xs[nt][e & 1], acc[r][nt][e]);
        }
      } else {
        uint4 b[NT][kSteps];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int64_t tok = tok0 + 8 * nt + g;
          const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + tok * p.x_row + col;
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const uint4 v = tok < p.tokens && col + 32 * s < p.k ? *reinterpret_cast<const uint4*>(x + 32 * s)
                                                                 : make_uint4(0, 0, 0, 0);
            // columns in the order of codes_bf16: (0, 2) (4, 6) (1, 3) (5, 7)
            b[nt][s] = make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.z, v.w, 0x5410),
                                  __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x7632));
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float d[NT][4] = {};
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            const uint32_t lo = cur.word(r, gi * kSteps + s, 0), hi = cur.word(r, gi * kSteps + s, 1);
            const uint32_t a0 = codes_bf16<0>(lo), a1 = codes_bf16<0>(hi), a2 = codes_bf16<1>(lo),
                           a3 = codes_bf16<1>(hi), a4 = codes_bf16<2>(lo), a5 = codes_bf16<2>(hi),
                           a6 = codes_bf16<3>(lo), a7 = codes_bf16<3>(hi);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_bf16_16816(d[nt], a0, a1, a2, a3, b[nt][s].x, b[nt][s].y);
              mma_bf16_16816(d[nt], a4, a5, a6, a7, b[nt][s].z, b[nt][s].w);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][nt][e] = fmaf(d[nt][e], cur.scale(gi, r, e >> 1), acc[r][nt][e]);
        }
      }
    }
  }

  float* mine = red + warp * kTok * kRedStride;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mine[(8 * nt + 2 * t + (e & 1)) * kRedStride + 16 * r + g + 8 * (e >> 1)] = acc[r][nt][e];
  __syncthreads();
  const int live = min(kTok, p.tokens - tok0) * kTileRows;
  float* part = red + kWarps * kTok * kRedStride;
  for (int i = threadIdx.x; i < live; i += kWarps * 32) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += red[(w * kTok + i / kTileRows) * kRedStride + i % kTileRows];
    if (p.splits > 1) {
      part[i] = sum;
    } else {
      const int row = tile * kTileRows + i % kTileRows;
      if (row < p.n) {
        if (p.bias) sum += __bfloat162float(p.bias[row]);
        p.y[(int64_t)(tok0 + i / kTileRows) * p.y_row + row] = __float2bfloat16_rn(sum);
      }
    }
  }
  if (p.splits > 1) {
    cluster_sync_all();  // every split has published its sums
    const uint32_t base = smem_u32(part);
    const int rank = (int)cluster_rank();
    for (int i = rank * (kWarps * 32) + threadIdx.x; i < live; i += p.splits * kWarps * 32) {
      float sum = 0.f;
      for (int s = 0; s < p.splits; ++s) sum += dsmem_ld(dsmem_map(base, s) + i * 4);
      const int row = tile * kTileRows + i % kTileRows;
      if (row < p.n) {
        if (p.bias) sum += __bfloat162float(p.bias[row]);
        p.y[(int64_t)(tok0 + i / kTileRows) * p.y_row + row] = __float2bfloat16_rn(sum);
      }
    }
    cluster_sync_all();  // the sums stay readable until every CTA has read them
  }
}

constexpr int skinny_smem(int nt) { return (kWarps * 8 * nt * kRedStride + 8 * nt * kTileRows) * 4; }

struct Dev {
  int sms = 0;
};
Dev g_dev[64];
std::mutex g_mu;

template <bool INT8, int G>
cudaError_t allow_smem() {
  cudaError_t e = cudaFuncSetAttribute(w4_skinny_kernel<INT8, G, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       skinny_smem(1));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(w4_skinny_kernel<INT8, G, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             skinny_smem(2));
  return e;
}

int device(int* sms) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LKV_ERR_CUDA;
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_dev[dev].sms == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return LKV_ERR_CUDA;
    if (allow_smem<true, 32>() != cudaSuccess || allow_smem<true, 64>() != cudaSuccess ||
        allow_smem<true, 128>() != cudaSuccess || allow_smem<false, 32>() != cudaSuccess ||
        allow_smem<false, 64>() != cudaSuccess || allow_smem<false, 128>() != cudaSuccess)
      return LKV_ERR_CUDA;
    g_dev[dev].sms = n;
  }
  *sms = g_dev[dev].sms;
  return LKV_OK;
}

// Splits of k over a cluster (a power of two <= 8): the fewest rounds of blocks per warp
// over the waves of CTAs, a round's worth for a CTA's start and end.
int choose_splits(int64_t ctas, int kblocks, int slots) {
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int s = 1; s <= 8 && s <= kblocks; s *= 2) {
    const int64_t waves = (ctas * s + slots - 1) / slots;
    const int per_warp = ((kblocks + s - 1) / s + kWarps - 1) / kWarps;
    const int64_t cost = waves * (2 * per_warp + 2) + (s > 1 ? 1 : 0);
    if (cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

template <bool INT8, int G, int NT>
int launch_skinny(const SkinnyParams& p, int tiles, cudaStream_t stream) {
  const dim3 grid(tiles, p.splits, (p.tokens + 8 * NT - 1) / (8 * NT));
  return launch_pdl_cluster(w4_skinny_kernel<INT8, G, NT>, grid, dim3(kWarps * 32), skinny_smem(NT), stream,
                            dim3(1, p.splits, 1), p) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

template <bool INT8, int G>
int skinny(const SkinnyParams& p, int tiles, cudaStream_t stream) {
  return p.tokens <= 8 ? launch_skinny<INT8, G, 1>(p, tiles, stream) : launch_skinny<INT8, G, 2>(p, tiles, stream);
}

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
      (reinterpret_cast<uintptr_t>(scales) & 1) || codes_row < k / 2 || scales_row < (k + group - 1) / group)
    return LKV_ERR_INVALID_ARGUMENT;
  const int64_t kblocks = (k + kTileK - 1) / kTileK, blocks = (n + kTileRows - 1) / kTileRows * kblocks;
  if (blocks > 0x7fffffff) return LKV_ERR_UNSUPPORTED;
  w4_pack_kernel<<<(unsigned)blocks, 256, 0, stream>>>(codes, codes_row, static_cast<const __nv_bfloat16*>(scales),
                                                       scales_row, n, k, group, kblocks,
                                                       static_cast<uint8_t*>(packed));
  return cudaGetLastError() == cudaSuccess ? LKV_OK : LKV_ERR_CUDA;
}

int w4_linear(const W4Args& a, cudaStream_t stream) {
  if (a.group != 32 && a.group != 64 && a.group != 128) return LKV_ERR_UNSUPPORTED;
  if (!shape_ok(a.n, a.k) || a.tokens < 0 || a.tokens > 0xfffff) return LKV_ERR_INVALID_ARGUMENT;
  if (a.tokens == 0) return LKV_OK;
  const bool int8 = a.x_scale != nullptr;
  const int align = int8 ? 8 : 16, elem = int8 ? 1 : 2;
  if (!a.x || !a.packed || !a.y || (reinterpret_cast<uintptr_t>(a.packed) & 15) ||
      (reinterpret_cast<uintptr_t>(a.x) % align) || (a.x_row * elem) % align || a.x_row < a.k || a.y_row < a.n ||
      (int8 && a.x_scale_row < (a.k + a.group - 1) / a.group))
    return LKV_ERR_INVALID_ARGUMENT;
  int sms = 0;
  const int st = device(&sms);
  if (st != LKV_OK) return st;
  if (a.tokens > kSkinnyTokens && w4_tile_aligned(a)) return w4_tile(a, sms, stream);
  const int tiles = (int)((a.n + kTileRows - 1) / kTileRows);
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
  const int64_t ztiles = a.tokens <= 8 ? 1 : (a.tokens + 15) / 16;
  p.splits = choose_splits(tiles * ztiles, p.kblocks, 2 * sms);
  if (int8)
    return a.group == 32   ? skinny<true, 32>(p, tiles, stream)
           : a.group == 64 ? skinny<true, 64>(p, tiles, stream)
                           : skinny<true, 128>(p, tiles, stream);
  return a.group == 32   ? skinny<false, 32>(p, tiles, stream)
         : a.group == 64 ? skinny<false, 64>(p, tiles, stream)
                         : skinny<false, 128>(p, tiles, stream);
}

}  // namespace lkv
