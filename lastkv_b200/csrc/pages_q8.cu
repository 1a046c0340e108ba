// Pages of a bf16 pool to 8 bits and back, and copies of whole pages (sm_100a).
//
//   quantise    per (page, KV head, keys or values, 8 tokens): s = max|x| / 127 and q = rne(x / s) in
//               fp32 arithmetic (zeros where s = 0); a block that holds an infinity or a NaN gets that scale and
//               zeros, so its values are NaN.  Tokens past the page's count are zeros and do not
//               count for the scale.
//   dequantise  bf16(q * s), or (staging for the prefill kernel) the codes themselves, which are
//               whole numbers up to 127 and exact in bf16 (keys) and f16 (values).
//   reorder     pages[dst[i]] = pages[src[i]] for all i at once, in several pools and layers.
// All three read and write each byte once and are bound by HBM.

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "pages_q8.cuh"

namespace lkv {

namespace {

constexpr int kWarps = 4;

struct QuantParams {
  const __nv_bfloat16* pool[2];  // keys, values
  int64_t pool_pages;
  const int32_t* pages;
  const int32_t* tokens;  // or null: 16
  uint8_t* codes;
  float* scales;
  int64_t q8_pages;
  const int32_t* out_pages;
  int64_t n;
  int hkv;
  int* err;
};

// A lane holds two rows (tokens 2p and 2p + 1) of one 16-column tile, so that every 4-byte word of the
// operand order is made in registers: 8 words per row pair, one of each of 4 column pairs x 2 rows for
// keys, of 8 columns for values.  They reach the order of memory through shared memory, word (tile t,
// row half h, g, c) at the place below: 16-byte vectors of (t & 1, h), which lane 4g + c reads.  The
// gaps and exclusive ors keep a warp's stores of one word on 32 banks.
template <int D>
struct Words {
  static constexpr int TILES = D / 16;
  static constexpr int PAIRS = 32 / TILES;  // row pairs per pass over the lanes
  static constexpr int PASSES = 8 / PAIRS;
  static constexpr int COUNT = D / 32 * 144;
  __device__ static int vector(int t2, int g, int c) { return t2 * 144 + g * 16 + ((c ^ (g >> 1)) * 4); }
  __device__ static int at(int t, int h, int g, int c) {
    return vector(t >> 1, g, c) + (((t & 1) * 2 + h) ^ (t >> 2));
  }
};

__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b) {  // |bf16| pairs, NaN stays
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
  return d;
}

__device__ __forceinline__ void load_tile_row(uint32_t (&v)[8], const __nv_bfloat16* at) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(at)), b = __ldg(reinterpret_cast<const uint4*>(at) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// One warp per (page, head, keys or values).  4096 pages of 8 heads of 128 (403 MB moved): 65-67 us, 6.0-6.2 TB/s,
// so HBM bounds it; a byte tile in shared memory and bf16 maxima one by one were issue-bound at 85.
// 64 wide: 41 us, 5.0 TB/s (a warp has 2 KB to read there, and starts and ends cost as much).
template <int D>
__global__ void __launch_bounds__(kWarps * 32, 8) quantise_pages_kernel(const QuantParams p) {
  using W = Words<D>;
  __shared__ __align__(16) uint32_t words_all[kWarps][W::COUNT];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
  if (item >= p.n * p.hkv * 2) return;
  const int which = (int)(item & 1), hk = (int)((item >> 1) % p.hkv);
  const int64_t n = (item >> 1) / p.hkv;
  const int64_t src = p.pages[n], dst = p.out_pages[n];
  if (src < 0 || src >= p.pool_pages || dst < 0 || dst >= p.q8_pages) {
    if (lane == 0 && hk == 0) report_error(p.err, DEVERR_BAD_PAGE, 8, (int)(src < 0 || src >= p.pool_pages ? src : dst));
    return;
  }
  const int valid = p.tokens ? min(max(p.tokens[n], 0), kPageTokens) : kPageTokens;
  const __nv_bfloat16* base = (which ? p.pool[1] : p.pool[0]) + (src * kPageTokens * p.hkv + hk) * D;
  const int64_t row_stride = (int64_t)p.hkv * D;
  const int t = lane % W::TILES, pair0 = lane / W::TILES;
  uint32_t v[W::PASSES][2][8];
#pragma unroll
  for (int i = 0; i < W::PASSES; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * (i * W::PAIRS + pair0) + e;
      if (r < valid) {
        load_tile_row(v[i][e], base + r * row_stride + t * 16);
      } else {
#pragma unroll
        for (int x = 0; x < 8; ++x) v[i][e][x] = 0;
      }
    }
  uint32_t* words = words_all[warp];
  float scales[W::PASSES];
#pragma unroll
  for (int i = 0; i < W::PASSES; ++i) {
    const int pair = i * W::PAIRS + pair0, h = pair >> 2, c0 = pair & 3;
    uint32_t m2 = 0;
#pragma unroll
    for (int x = 0; x < 16; ++x) m2 = abs_max2(m2, v[i][x >> 3][x & 7]);
#pragma unroll
    for (int o = 2 * W::TILES; o > 0; o >>= 1) m2 = abs_max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    const float amax = max_nan(bf16_lo(m2), bf16_hi(m2));
    const float scale = amax / 127.0f;
    scales[i] = scale;
    // The code is the fp32 quotient x / scale rounded to nearest even, by two divisions per block: x * inv with
    // inv = 127 / max, rounded by the addition that puts q + 128 into the low byte of 1.5 * 2^23 + 128 + q.  A bf16 x
    // comes closer than 2^-17 to a place half way between two codes only where 127 x / max is one; but for
    // x = max / 2, at 63.5, the scale and inv are exact there.  So it is enough that max / 2 goes to the side that its
    // quotient is on (64 from 63.5 on): inv is one step from the nearest where that one goes to the other side.
    float inv = 127.0f / amax;
    {
      const bool up = 0.5f * amax / scale >= 63.5f, inv_up = fmaf(amax, inv, -127.0f) >= 0.f;  // (the latter exact)
      if (up != inv_up) inv = __uint_as_float(__float_as_uint(inv) + (up ? 1u : ~0u));
    }
    if (!(amax >= 1e-30f && amax < INFINITY)) {
      // scales with few bits, or none, or not finite: the codes themselves take the values' place
      const bool zero = !(amax < INFINITY) || scale == 0.f;
      auto code = [&](float x) { return zero ? 0.f : rintf(x / scale); };
      inv = 1.f;
#pragma unroll 1
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t w = e ? v[i][1][x] : v[i][0][x];
          const uint32_t c = pack_bf16(code(bf16_lo(w)), code(bf16_hi(w)));
          if (e) v[i][1][x] = c;
          else v[i][0][x] = c;
        }
    }
    auto codes = [&](uint32_t w) {
      return __ffma2_rn(make_float2(bf16_lo(w), bf16_hi(w)), make_float2(inv, inv),
                        make_float2(12583040.0f, 12583040.0f));
    };
    auto word = [](float a, float b, float c, float d) {
      return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                         __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
    };
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // columns 2x, 2x + 1, 2x + 8 and 2x + 9
      const float2 a0 = codes(v[i][0][x]), a8 = codes(v[i][0][x + 4]);
      const float2 b0 = codes(v[i][1][x]), b8 = codes(v[i][1][x + 4]);
      if (which == 0) {
        words[W::at(t, h, 2 * c0, x)] = word(a0.x, a8.x, a0.y, a8.y);
        words[W::at(t, h, 2 * c0 + 1, x)] = word(b0.x, b8.x, b0.y, b8.y);
      } else {
        words[W::at(t, h, 2 * x, c0)] = word(a0.x, a8.x, b0.x, b8.x);
        words[W::at(t, h, 2 * x + 1, c0)] = word(a0.y, a8.y, b0.y, b8.y);
      }
    }
  }
  __syncwarp();
  const int64_t block = dst * p.hkv + hk;
  uint8_t* out = p.codes + (block * 2 + which) * 16 * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint4 w = *reinterpret_cast<const uint4*>(words + W::vector(i, lane >> 2, lane & 3));
    if (i & 2) w = make_uint4(w.y, w.x, w.w, w.z);
    *reinterpret_cast<uint4*>(out + i * 512 + lane * 16) = w;
  }
  if constexpr (W::PASSES == 2) {
    if (lane == 0)
      *reinterpret_cast<float2*>(p.scales + block * kScalesPerBlock + 2 * which) = make_float2(scales[0], scales[1]);
  } else {
    if (lane % 16 == 0) p.scales[block * kScalesPerBlock + 2 * which + lane / 16] = scales[0];
  }
}

struct DequantParams {
  const uint8_t* codes;
  const float* scales;
  int64_t q8_pages;
  __nv_bfloat16* pool[2];
  int64_t pool_pages;
  int hkv;
  int* err;
  // a list of pages
  const int32_t* pages;
  const int32_t* out_pages;
  int64_t n;
  // or the `columns` leading ones of block tables: row b's column j becomes page b * width + j
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* num_q8;  // or null: every column
  const int32_t* seq_k;
  int batch, W, width, columns;
};

// Back to rows of bf16, one warp per (page, head, keys or values), through a byte tile in shared memory:
// rows of D + 16 bytes, so that whole 16-byte pieces of a row are written (words made in registers as
// above, which would write rows in pieces of half a sector, took 9.4 us where this takes 8.0).  4096 pages
// of 8 heads of 128: 67 us, 6.0 TB/s; 64 wide: 37 us, 5.4 TB/s.
// STAGE: the codes themselves, keys in bf16 and values in f16 (the prefill kernel applies the scales); where a scale is not finite
// the keys are NaN, so that the tokens' scores are, and the values zero.
template <int D, bool STAGE>
__global__ void __launch_bounds__(kWarps * 32) dequantise_pages_kernel(const DequantParams p) {
  constexpr int PITCH = D + 16;
  constexpr int LANES = D / 8, STEP = 32 / LANES, LOADS = 16 / STEP;
  __shared__ __align__(16) uint8_t tile_all[kWarps][16 * PITCH];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
  const int which = (int)(item & 1), hk = (int)((item >> 1) % p.hkv);
  const int64_t n = (item >> 1) / p.hkv;
  int64_t src, dst;
  if constexpr (STAGE) {
    const int b = (int)(n / p.columns), j = (int)(n % p.columns);
    if (b >= p.batch) return;
    const int pages = min((max(p.seq_k[b], 0) + kPageTokens - 1) / kPageTokens, p.W);
    if (j >= (p.num_q8 ? min(p.num_q8[b], pages) : pages)) return;
    src = p.bt[(int64_t)b * p.bt_stride + j];
    dst = (int64_t)b * p.width + j;
  } else {
    if (n >= p.n) return;
    src = p.pages[n];
    dst = p.out_pages[n];
  }
  if (src < 0 || src >= p.q8_pages || dst < 0 || dst >= p.pool_pages) {
    const bool bad_src = src < 0 || src >= p.q8_pages;
    if (lane == 0 && hk == 0) report_error(p.err, DEVERR_BAD_PAGE, 9, (int)(bad_src ? src : dst));
    if (!STAGE) return;
  }
  const bool have = src >= 0 && src < p.q8_pages;  // a staged page that is not there reads as zeros
  const int g = lane >> 2, c = lane & 3;
  const int64_t block = src * p.hkv + hk;
  const uint8_t* in = p.codes + (block * 2 + which) * 16 * D;
  uint8_t* tile = tile_all[warp];
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  uint4 v[D / 32];
  if (have) s = *reinterpret_cast<const float4*>(p.scales + block * kScalesPerBlock);
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    v[i] = have ? __ldcs(reinterpret_cast<const uint4*>(in + i * 512 + lane * 16)) : make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int t = 2 * i + (x >> 1), h = x & 1;
      if (which == 0) {
        uint8_t* at = tile + (8 * h + g) * PITCH + 16 * t + 2 * c;
        *reinterpret_cast<uint16_t*>(at) = (uint16_t)__byte_perm(w[x], 0, 0x4420);
        *reinterpret_cast<uint16_t*>(at + 8) = (uint16_t)__byte_perm(w[x], 0, 0x4431);
      } else {
        uint8_t* at = tile + (8 * h + 2 * c) * PITCH + 16 * t + g;
        at[0] = (uint8_t)w[x];
        at[8] = (uint8_t)(w[x] >> 8);
        at[PITCH] = (uint8_t)(w[x] >> 16);
        at[PITCH + 8] = (uint8_t)(w[x] >> 24);
      }
    }
  }
  __syncwarp();
  const float s0 = which ? s.z : s.x, s1 = which ? s.w : s.y;
  // staged keys of tokens whose keys or values have a scale that is not finite
  const bool bad0 = !(fabsf(s.x) < INFINITY) || !(fabsf(s.z) < INFINITY);
  const bool bad1 = !(fabsf(s.y) < INFINITY) || !(fabsf(s.w) < INFINITY);
  __nv_bfloat16* base = (which ? p.pool[1] : p.pool[0]) + (dst * kPageTokens * p.hkv + hk) * D;
  const int64_t row_stride = (int64_t)p.hkv * D;
  // staged values of blocks whose scale the prefill kernel takes as kMinValueScale: times what is missing (0 for 0, and
  // for whatever lies behind a row's end)
  const float v0 = fminf(fmaxf(s0 * 0x1p90f, 0.f), 1.f), v1 = fminf(fmaxf(s1 * 0x1p90f, 0.f), 1.f);
  const int r0 = lane / LANES, col = (lane % LANES) * 8;
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r = i * STEP + r0;
    const uint2 q = *reinterpret_cast<const uint2*>(tile + r * PITCH + col);
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = (e & 2) ? q.y : q.x;
      const uint32_t two = w >> ((e & 1) * 16);
      const float a = (float)((int)(two & 255u) - 128), b = (float)((int)(two >> 8 & 255u) - 128);
      if constexpr (STAGE) {
        const float v = r < 8 ? v0 : v1;
        o[e] = which ? pack_f16(a * v, b * v) : (r < 8 ? bad0 : bad1) ? 0x7fff7fffu : pack_bf16(a, b);
      } else {
        const float sc = r < 8 ? s0 : s1;
        o[e] = pack_bf16(a * sc, b * sc);
      }
    }
    *reinterpret_cast<uint4*>(base + r * row_stride + col) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---------------------------------------------------------------- copies of pages

constexpr int kMaxPools = 8, kMaxCopies = 2048;
constexpr int kCopyThreads = 128;
constexpr int kCopyBytes = 64 * 1024, kSliceBytes = 2048;

struct ReorderParams {
  uint8_t* pool[kMaxPools];
  int64_t page_bytes[kMaxPools];
  int64_t pages[kMaxPools];
  int64_t first_slice[kMaxPools + 1];  // slices of one layer, pool after pool
  const int32_t* src;
  const int32_t* dst;
  int n, slice_bytes;
  int64_t layer_stride, id_limit;
  int* err;
};

// A CTA moves the same slice of every listed page of one pool and layer by bulk copies through shared
// memory: all of them are read before any is written, so the lists may permute pages among themselves.
// Slices are as wide as 64 KB over the list allow, up to 2 KB; three such CTAs fit an SM, so one's reads
// run beside another's writes.  64 rows of 32 layers (8 heads of 128, 268 MB moved): 45 us, 6.0 TB/s
// (through registers, with 512 bytes a page in flight: 58); 4 rows of 12 layers (12 heads of 64): 2.6 us.
__global__ void __launch_bounds__(kCopyThreads) reorder_pages_kernel(const ReorderParams p) {
  extern __shared__ __align__(128) uint8_t held[];
  __shared__ uint64_t loaded;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    mbar_init(&loaded, kCopyThreads);
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  const int64_t slice = blockIdx.x;
  int pool = 0;
  while (slice >= p.first_slice[pool + 1]) ++pool;
  const int64_t first = blockIdx.y * p.layer_stride, page_bytes = p.page_bytes[pool], pages = p.pages[pool];
  const int64_t at = (slice - p.first_slice[pool]) * p.slice_bytes;
  const uint32_t bytes = (uint32_t)min((int64_t)p.slice_bytes, page_bytes - at);
  uint8_t* base = p.pool[pool] + at;
  // with several layers an id is one of a layer's pages, so no layer writes what another reads
  auto bad = [&](int id) { return id < 0 || id >= p.id_limit || id + first >= pages; };
  uint32_t expected = 0;
  for (int r = threadIdx.x; r < p.n; r += kCopyThreads) {
    const int s = p.src[r], d = p.dst[r];
    if (bad(s) || bad(d)) {
      if (at == 0) report_error(p.err, DEVERR_BAD_PAGE, 10, bad(s) ? s : d);
    } else if (s != d) {
      expected += bytes;
    }
  }
  mbar_arrive_expect_tx(&loaded, expected);
  for (int r = threadIdx.x; r < p.n; r += kCopyThreads) {
    const int s = p.src[r], d = p.dst[r];
    if (!bad(s) && !bad(d) && s != d)
      bulk_load(held + (size_t)r * p.slice_bytes, base + (s + first) * page_bytes, bytes, &loaded);
  }
  if (!mbar_wait(&loaded, 0)) {
    report_error(p.err, DEVERR_WAIT_TIMEOUT, 10, (int)slice);
    mbar_wait(&loaded, 0);
    return;
  }
  for (int r = threadIdx.x; r < p.n; r += kCopyThreads) {
    const int s = p.src[r], d = p.dst[r];
    if (!bad(s) && !bad(d) && s != d)
      bulk_store(base + (d + first) * page_bytes, held + (size_t)r * p.slice_bytes, bytes);
  }
  bulk_commit_group();
  bulk_wait_group_read0();  // shared memory is released when the CTA exits
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

int check_pages(const void* pool_k, const void* pool_v, int64_t pool_pages, const void* codes, const void* scales,
                int64_t q8_pages, int hkv, int d) {
  if (d != 64 && d != 128) return LKV_ERR_UNSUPPORTED;
  if (hkv < 1 || hkv > 256 || pool_pages < 0 || q8_pages < 0 || pool_pages > INT32_MAX || q8_pages > INT32_MAX)
    return LKV_ERR_INVALID_ARGUMENT;
  if (!pool_k || !pool_v || !codes || !scales) return LKV_ERR_INVALID_ARGUMENT;
  if (misaligned(pool_k, 16) || misaligned(pool_v, 16) || misaligned(codes, 16) || misaligned(scales, 16))
    return LKV_ERR_INVALID_ARGUMENT;
  return LKV_OK;
}

}  // namespace

int quantise_pages(const void* pool_k, const void* pool_v, int64_t pool_pages, const int32_t* pages,
                   const int32_t* tokens, void* codes, float* scales, int64_t q8_pages, const int32_t* out_pages,
                   int64_t n, int hkv, int d, int* err, cudaStream_t stream) {
  const int st = check_pages(pool_k, pool_v, pool_pages, codes, scales, q8_pages, hkv, d);
  if (st != LKV_OK) return st;
  if (n < 0 || (n > 0 && (!pages || !out_pages))) return LKV_ERR_INVALID_ARGUMENT;
  if (n == 0) return LKV_OK;
  QuantParams p{};
  p.pool[0] = static_cast<const __nv_bfloat16*>(pool_k);
  p.pool[1] = static_cast<const __nv_bfloat16*>(pool_v);
  p.pool_pages = pool_pages;
  p.pages = pages;
  p.tokens = tokens;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = scales;
  p.q8_pages = q8_pages;
  p.out_pages = out_pages;
  p.n = n;
  p.hkv = hkv;
  p.err = err;
  const int64_t blocks = (n * hkv * 2 + kWarps - 1) / kWarps;
  if (n > INT32_MAX || blocks > INT32_MAX) return LKV_ERR_UNSUPPORTED;
  const auto kern = d == 128 ? quantise_pages_kernel<128> : quantise_pages_kernel<64>;
  return launch_pdl(kern, dim3((unsigned)blocks), dim3(kWarps * 32), 0, stream, p) == cudaSuccess ? LKV_OK
                                                                                                  : LKV_ERR_CUDA;
}

namespace {
int launch_dequantise(const DequantParams& p, int64_t n, int d, bool stage, cudaStream_t stream) {
  const int64_t blocks = (n * p.hkv * 2 + kWarps - 1) / kWarps;
  if (n > INT32_MAX || blocks > INT32_MAX) return LKV_ERR_UNSUPPORTED;
  const auto kern = d == 128 ? (stage ? dequantise_pages_kernel<128, true> : dequantise_pages_kernel<128, false>)
                             : (stage ? dequantise_pages_kernel<64, true> : dequantise_pages_kernel<64, false>);
  return launch_pdl(kern, dim3((unsigned)blocks), dim3(kWarps * 32), 0, stream, p) == cudaSuccess ? LKV_OK
                                                                                                  : LKV_ERR_CUDA;
}
}  // namespace

int dequantise_pages(const void* codes, const float* scales, int64_t q8_pages, const int32_t* pages, void* pool_k,
                     void* pool_v, int64_t pool_pages, const int32_t* out_pages, int64_t n, int hkv, int d, int* err,
                     cudaStream_t stream) {
  const int st = check_pages(pool_k, pool_v, pool_pages, codes, scales, q8_pages, hkv, d);
  if (st != LKV_OK) return st;
  if (n < 0 || (n > 0 && (!pages || !out_pages))) return LKV_ERR_INVALID_ARGUMENT;
  if (n == 0) return LKV_OK;
  DequantParams p{};
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = scales;
  p.q8_pages = q8_pages;
  p.pool[0] = static_cast<__nv_bfloat16*>(pool_k);
  p.pool[1] = static_cast<__nv_bfloat16*>(pool_v);
  p.pool_pages = pool_pages;
  p.hkv = hkv;
  p.err = err;
  p.pages = pages;
  p.out_pages = out_pages;
  p.n = n;
  return launch_dequantise(p, n, d, false, stream);
}

int stage_pages(const void* codes, const float* scales, int64_t q8_pages, const int32_t* bt, int64_t bt_stride,
                const int32_t* num_q8, const int32_t* seq_k, int batch, int W, void* stage_k, void* stage_v, int width,
                int hkv, int d, int* err, cudaStream_t stream) {
  if (batch < 0 || W < 0 || width < 0) return LKV_ERR_INVALID_ARGUMENT;
  const int columns = std::min(width, W);
  if (batch == 0 || columns == 0) return LKV_OK;
  const int st = check_pages(stage_k, stage_v, (int64_t)batch * width, codes, scales, q8_pages, hkv, d);
  if (st != LKV_OK) return st;
  if (!bt || !seq_k) return LKV_ERR_INVALID_ARGUMENT;
  DequantParams p{};
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = scales;
  p.q8_pages = q8_pages;
  p.pool[0] = static_cast<__nv_bfloat16*>(stage_k);
  p.pool[1] = static_cast<__nv_bfloat16*>(stage_v);
  p.pool_pages = (int64_t)batch * width;
  p.hkv = hkv;
  p.err = err;
  p.bt = bt;
  p.bt_stride = bt_stride;
  p.num_q8 = num_q8;
  p.seq_k = seq_k;
  p.batch = batch;
  p.W = W;
  p.width = width;
  p.columns = columns;
  return launch_dequantise(p, (int64_t)batch * columns, d, true, stream);
}

int reorder_pages(void* const* pools, const int64_t* page_bytes, const int64_t* pages, int num_pools,
                  const int32_t* src, const int32_t* dst, int n, int layers, int64_t layer_stride, int* err,
                  cudaStream_t stream) {
  if (num_pools < 1 || num_pools > kMaxPools || !pools || !page_bytes || !pages) return LKV_ERR_INVALID_ARGUMENT;
  if (n < 0 || layers < 0 || layer_stride < 0 || (n > 0 && (!src || !dst))) return LKV_ERR_INVALID_ARGUMENT;
  if (n > kMaxCopies || layers > 65535) return LKV_ERR_UNSUPPORTED;
  if (layers > 1 && (layer_stride < 1 || layer_stride > INT32_MAX)) return LKV_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < num_pools; ++i)
    if (!pools[i] || misaligned(pools[i], 16) || page_bytes[i] < 16 || page_bytes[i] % 16 || pages[i] < 1)
      return LKV_ERR_INVALID_ARGUMENT;
  if (n == 0 || layers == 0) return LKV_OK;
  ReorderParams p{};
  p.src = src;
  p.dst = dst;
  p.n = n;
  p.layer_stride = layer_stride;
  p.id_limit = layers > 1 ? layer_stride : (int64_t)INT32_MAX + 1;
  p.err = err;
  p.slice_bytes = 16;
  while (p.slice_bytes < kSliceBytes && (int64_t)n * p.slice_bytes * 2 <= kCopyBytes) p.slice_bytes *= 2;
  int64_t slices = 0;
  for (int i = 0; i < num_pools; ++i) {
    p.pool[i] = static_cast<uint8_t*>(pools[i]);
    p.page_bytes[i] = page_bytes[i];
    p.pages[i] = pages[i];
    p.first_slice[i] = slices;
    slices += (page_bytes[i] + p.slice_bytes - 1) / p.slice_bytes;
  }
  for (int i = num_pools; i <= kMaxPools; ++i) p.first_slice[i] = slices;
  if (slices > INT32_MAX) return LKV_ERR_UNSUPPORTED;
  const int smem = n * p.slice_bytes;
  if (cudaFuncSetAttribute(reorder_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCopyBytes) != cudaSuccess)
    return LKV_ERR_CUDA;
  return launch_pdl(reorder_pages_kernel, dim3((unsigned)slices, (unsigned)layers), dim3(kCopyThreads), smem, stream, p) ==
                 cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

}  // namespace lkv
