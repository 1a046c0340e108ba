// Beam search's selection over beams and vocabulary (sm_100a).
//
// For batch item b with K beams, scores c[k] and rows of logits x[k][V]:
//     total[k][v] = c[k] + x[k][v] - log sum_u exp x[k][u]
// and the `select` largest totals of the K * V, largest first, equal ones in the order of k * V + v.
// A finished beam has one candidate, its end token at its score.  Totals are compared in 64 bits.
// Within a beam they are ordered as its logits are, so one pass over the logits in their own type
// finds each row's `select` largest together with its maximum and sum of exponentials (fp32):
//
//   beam_rows    A CTA takes a stretch of a row in tiles of 8192 values, 32 in each thread's
//                registers.  It keeps the stretch's best `select` as sorted 64-bit keys (the value as
//                an ordered integer, then the complement of the index, so that no two are equal) and
//                collects what beats the last of them.  A tile with too many such values (the first
//                one) first raises the bar to a key that at least `select` of its values reach: the
//                select-th largest of a warp's 32 lane maxima, in the warp where that is largest, or
//                the (select / 8)-th, in the warp where it is least.  If still too many pass, the
//                tile's best are taken out one by one.
//   beam_merge   A CTA per batch item joins each row's stretches, then the rows: lists are sorted, so a
//                candidate's rank is a sum of binary searches.
//
// Bound by HBM for many rows and by two launches for few.

#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace lkv {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPer = 32;                 // values per thread and tile
constexpr int kTile = kThreads * kPer;   // 8192
constexpr int kMaxSelect = 32;
constexpr int kMaxBeams = 64;
constexpr int kCandidates = 1024;        // a tile's values over the bar
constexpr int kMaxStretches = 64;
constexpr float kLog2e = 1.4426950408889634f;

// Keys of equal order: a larger value is a larger key, -0 equals 0, a NaN counts as -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t max_key(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max_key(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}

struct RowsParams {
  const void* logits;
  int64_t row_stride;
  int64_t V;
  const uint8_t* finished;  // [rows] or null
  int64_t eos;
  int select, stretches, tiles_per;
  uint64_t* keys;  // [rows][stretches][select], sorted, 0 past the last
  float2* sums;    // [rows][stretches]: maximum, sum of exp(x - maximum)
};

template <typename T>
__global__ void __launch_bounds__(kThreads) beam_rows_kernel(const RowsParams p) {
  constexpr int VE = 16 / sizeof(T);  // values per 16-byte load
  __shared__ uint64_t cand[kCandidates + kMaxSelect];
  __shared__ uint64_t best[2][kMaxSelect];
  __shared__ uint64_t warp_key[kWarps], warp_eighth[kWarps];
  __shared__ float2 warp_sum[kWarps];
  __shared__ int count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.y;
  const int n = p.select;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  // tiles start at 16-byte boundaries, so a row's first may begin before it
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const bool done = p.finished && p.finished[row];
  const int64_t first = (int64_t)blockIdx.x * p.tiles_per;
  int cur = 0;
  if (tid < n) best[0][tid] = 0;
  float m = -INFINITY, sum = 0.f;
  for (int64_t t = first; t < first + p.tiles_per; ++t) {
    const int64_t base = t * kTile - lead;
    if (base >= p.V) break;
    float v[kPer];
    // the index of v[e]: base + (e / VE * kThreads + tid) * VE + e % VE
    auto index = [&](int e) { return base + (int64_t)(e / VE * kThreads + tid) * VE + e % VE; };
    auto inside = [&](int64_t i) { return i >= 0 && i < p.V; };
#pragma unroll
    for (int i = 0; i < kPer / VE; ++i) {
      const int64_t at = index(i * VE);
      if (done) {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[i * VE + e] = at + e == p.eos ? 0.f : -INFINITY;
      } else if (at >= 0 && at + VE <= p.V) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x + at));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if constexpr (sizeof(T) == 2) v[i * VE + e] = e & 1 ? bf16_hi(u[e / 2]) : bf16_lo(u[e / 2]);
          else v[i * VE + e] = __uint_as_float(u[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[i * VE + e] = inside(at + e) ? (float)x[at + e] : -INFINITY;
      }
    }
    const bool whole = base >= 0 && base + kTile <= p.V;
    // the thread's maximum and sum, over all its tiles; a NaN stays in the sum
    float top = v[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) top = fmaxf(top, v[e]);
    const float nm = fmaxf(m, top);
    if (nm != -INFINITY) {
      if (nm != m) sum *= exp2f((m - nm) * kLog2e);
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum += ex2_approx((v[e] - nm) * kLog2e);
      m = nm;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum = v[e] == v[e] ? sum : NAN;
    }
    auto key = [&](int e) -> uint64_t {
      const int64_t i = index(e);
      return whole || inside(i) ? (uint64_t)ordered(v[e]) << 32 | (0xffffffffu - (uint32_t)i) : 0;
    };
    __syncthreads();  // best[cur] is written; count and cand are free
    uint64_t bar = best[cur][n - 1] + 1;  // the least key that is worth collecting
    if (tid == 0) count = 0;
    // a first look, at the values' high words alone: most tiles after a stretch's first hold nothing
    const bool any = ordered(top) >= (uint32_t)(bar >> 32);
    if (!__syncthreads_or(any)) continue;
    int mine = 0;
    if (any) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) mine += key(e) >= bar;
    }
    if (mine) atomicAdd(&count, mine);
    __syncthreads();
    int total = count;
    if (total > kCandidates) {
      uint64_t big = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) big = max_key(big, key(e));
      int rank = 0;
      for (int l = 0; l < 32; ++l) {
        const uint64_t other = __shfl_sync(0xffffffffu, big, l);
        rank += other > big || (other == big && l < lane);
      }
      if (rank == n - 1) warp_key[warp] = big;
      if (rank == (n + kWarps - 1) / kWarps - 1) warp_eighth[warp] = big;
      __syncthreads();
      uint64_t least = warp_eighth[0];
      for (int w = 0; w < kWarps; ++w) {
        bar = max_key(bar, warp_key[w]);
        least = min(least, warp_eighth[w]);
      }
      bar = max_key(bar, least);
      if (tid == 0) count = 0;
      __syncthreads();
      mine = 0;
      if (big >= bar) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) mine += key(e) >= bar;
      }
      if (mine) atomicAdd(&count, mine);
      __syncthreads();
      total = count;
    }
    __syncthreads();  // count is read
    if (total <= kCandidates) {
      if (tid == 0) count = 0;
      __syncthreads();
      if (mine) {
        int at = atomicAdd(&count, mine);  // the order of the list does not matter: keys are ranked below
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const uint64_t k = key(e);
          if (k >= bar) cand[at++] = k;
        }
      }
    } else {
      // the tile's best, one after another
      uint64_t last = ~0ull;
      for (int r = 0; r < n; ++r) {
        uint64_t big = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const uint64_t k = key(e);
          if (k < last) big = max_key(big, k);
        }
        big = warp_max_key(big);
        if (lane == 0) warp_key[warp] = big;
        __syncthreads();
        big = warp_key[0];
        for (int w = 1; w < kWarps; ++w) big = max_key(big, warp_key[w]);
        if (tid == 0) cand[r] = big;
        last = big;
        __syncthreads();
      }
      total = n;
    }
    if (tid < n) {
      best[cur ^ 1][tid] = 0;
    }
    __syncthreads();
    // the new best: every entry of the old list and of the collected ones finds its rank among all
    if (tid < n) cand[total + tid] = best[cur][tid];
    __syncthreads();
    const int all = total + n;
    for (int a = tid; a < all; a += kThreads) {
      const uint64_t k = cand[a];
      if (k == 0) continue;
      int rank = 0;
      for (int b = 0; b < all; ++b) rank += cand[b] > k;
      if (rank < n) best[cur ^ 1][rank] = k;
    }
    cur ^= 1;
  }
  // the stretch's maximum and sum: warps, then the CTA, in a fixed order
  auto join = [](float2 a, float2 b) {
    const float t = fmaxf(a.x, b.x);
    if (t == -INFINITY) return make_float2(t, a.y + b.y);
    return make_float2(t, (a.x == t ? a.y : a.y * exp2f((a.x - t) * kLog2e)) +
                              (b.x == t ? b.y : b.y * exp2f((b.x - t) * kLog2e)));
  };
  float2 ms = make_float2(m, sum);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, ms.x, o), __shfl_xor_sync(0xffffffffu, ms.y, o));
    ms = lane & o ? join(other, ms) : join(ms, other);  // the same operands in both lanes' order
  }
  if (lane == 0) warp_sum[warp] = ms;
  __syncthreads();
  const int64_t at = row * p.stretches + blockIdx.x;
  if (tid == 0) {
    ms = warp_sum[0];
    for (int w = 1; w < kWarps; ++w) ms = join(ms, warp_sum[w]);
    p.sums[at] = ms;
  }
  if (tid < n) p.keys[at * n + tid] = best[cur][tid];
}

struct MergeParams {
  const uint64_t* keys;
  const float2* sums;
  const float* scores;  // [B, K]
  const uint8_t* finished;
  int64_t V, eos;
  int K, select, stretches;
  int rows_per_pass;  // rows whose keys fit in shared memory at once
  float* out_scores;
  int64_t* out_rows;
  int64_t* out_tokens;
  uint8_t* out_finished;
};

// How many of the n keys, sorted from the largest, are larger than k.
__device__ __forceinline__ int larger(const uint64_t* list, int n, uint64_t k) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] > k) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

constexpr int kMergeThreads = 512;

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const MergeParams p) {
  extern __shared__ uint64_t keys[];  // [rows_per_pass][stretches][select]
  // A total is (x - top) + norm: the maximum is taken off first, so that rows of values like a type's
  // lowest keep their sums' logarithms and their scores.  norm NaN: every total of the row is -inf.
  __shared__ double tops[kMaxBeams], norm[kMaxBeams];
  __shared__ double total[kMaxBeams * kMaxSelect];
  __shared__ uint32_t token[kMaxBeams * kMaxSelect];
  const int b = blockIdx.x, n = p.select, K = p.K, S = p.stretches, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  for (int k = tid; k < K; k += kMergeThreads) {
    const int64_t row = (int64_t)b * K + k;
    float top = -INFINITY;
    double sum = 0;
    for (int s = 0; s < S; ++s) top = fmaxf(top, p.sums[row * S + s].x);
    for (int s = 0; s < S; ++s) {
      const float2 ms = p.sums[row * S + s];
      if (ms.x == -INFINITY) sum += ms.y;  // 0, or a NaN
      else sum += (double)ms.y * (ms.x == top ? 1.0 : (double)expf(ms.x - top));
    }
    const bool done = p.finished && p.finished[row];
    const double c = (double)p.scores[row], rest = done ? 0.0 : log(sum);
    tops[k] = done ? 0.0 : (double)top;
    norm[k] = fabs(c) < INFINITY && fabs(tops[k]) < INFINITY && fabs(rest) < INFINITY ? c - rest : NAN;
  }
  for (int k0 = 0; k0 < K; k0 += p.rows_per_pass) {
    const int rows = min(p.rows_per_pass, K - k0), per = S * n;
    const uint64_t* in = p.keys + ((int64_t)b * K + k0) * per;
    __syncthreads();
    for (int i = tid; i < rows * per; i += kMergeThreads) keys[i] = in[i];
    __syncthreads();
    for (int i = tid; i < rows * per; i += kMergeThreads) {
      const uint64_t k = keys[i];
      if (k == 0) continue;
      const int r = i / per, s = i % per / n;
      int rank = i % n;
      const uint64_t* row = keys + r * per;
      for (int o = 0; o < S && rank < n; ++o)
        if (o != s) rank += larger(row + o * n, n, k);
      if (rank >= n) continue;
      const double c = norm[k0 + r];
      const double t = ((double)from_ordered((uint32_t)(k >> 32)) - tops[k0 + r]) + c;
      const bool alive = c == c;
      // all totals of a row without a finite score or sum are -inf: its first tokens, in their order
      total[(k0 + r) * n + rank] = alive && t == t ? t : -INFINITY;
      token[(k0 + r) * n + rank] = alive ? 0xffffffffu - (uint32_t)k : (uint32_t)rank;
    }
  }
  __syncthreads();
  for (int i = tid; i < K * n; i += kMergeThreads) {
    const int k = i / n;
    const double t = total[i];
    int rank = i % n;
    for (int o = 0; o < K && rank < n; ++o) {
      if (o == k) continue;
      // entries of row o that come before (t, k): larger, or equal and of an earlier row
      const double* list = total + o * n;
      int lo = 0, hi = n;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > t || (list[mid] == t && o < k)) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank >= n) continue;
    const int64_t row = (int64_t)b * K + k, at = (int64_t)b * n + rank;
    p.out_scores[at] = (float)t;
    p.out_rows[at] = row;
    p.out_tokens[at] = token[i];
    if (p.out_finished) p.out_finished[at] = (int64_t)token[i] == p.eos || (p.finished && p.finished[row]);
  }
}

struct Split {
  int stretches, tiles_per;
};
// About four CTAs per SM over all rows, whole tiles each.
Split split_rows(int64_t rows, int64_t V, int sms) {
  const int64_t tiles = (V + 7 + kTile - 1) / kTile;
  int64_t s = std::min<int64_t>({tiles, (int64_t)kMaxStretches, std::max<int64_t>(1, 4ll * sms / rows)});
  const int64_t per = (tiles + s - 1) / s;
  return {(int)((tiles + per - 1) / per), (int)per};
}

constexpr int kMergeSmem = 128 * 1024;

}  // namespace

size_t beam_workspace_bytes(int64_t rows, int select) {
  if (rows < 0 || select < 1) return 0;
  return (size_t)rows * kMaxStretches * ((size_t)select * sizeof(uint64_t) + sizeof(float2));
}

int beam_select(const void* logits, int64_t row_stride, int fp32, const float* scores, const uint8_t* finished,
                int64_t eos, int batch, int beams, int64_t vocab, int select, float* out_scores, int64_t* out_rows,
                int64_t* out_tokens, uint8_t* out_finished, void* workspace, size_t workspace_bytes,
                cudaStream_t stream) {
  if (batch < 0 || beams < 1 || vocab < 1 || select < 1 || select > vocab) return LKV_ERR_INVALID_ARGUMENT;
  if (beams > kMaxBeams || select > kMaxSelect || vocab > INT32_MAX) return LKV_ERR_UNSUPPORTED;
  if (batch == 0) return LKV_OK;
  const int64_t rows = (int64_t)batch * beams;
  if (rows > 65535) return LKV_ERR_UNSUPPORTED;
  if (!logits || !scores || !out_scores || !out_rows || !out_tokens) return LKV_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(logits) & (fp32 ? 3 : 1)) return LKV_ERR_INVALID_ARGUMENT;
  if (rows > 1 && row_stride < 0) return LKV_ERR_INVALID_ARGUMENT;
  if (finished && (eos < 0 || eos >= vocab)) return LKV_ERR_INVALID_ARGUMENT;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return LKV_ERR_CUDA;
  const Split sp = split_rows(rows, vocab, sms);
  const size_t entries = (size_t)rows * sp.stretches;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
      workspace_bytes < entries * (select * sizeof(uint64_t) + sizeof(float2)))
    return LKV_ERR_WORKSPACE;
  RowsParams r{};
  r.logits = logits;
  r.row_stride = row_stride;
  r.V = vocab;
  r.finished = finished;
  r.eos = eos;
  r.select = select;
  r.stretches = sp.stretches;
  r.tiles_per = sp.tiles_per;
  r.sums = static_cast<float2*>(workspace);
  r.keys = reinterpret_cast<uint64_t*>(r.sums + entries);
  const dim3 grid((unsigned)sp.stretches, (unsigned)rows);
  const auto kern = fp32 ? beam_rows_kernel<float> : beam_rows_kernel<__nv_bfloat16>;
  if (launch_pdl(kern, grid, dim3(kThreads), 0, stream, r) != cudaSuccess) return LKV_ERR_CUDA;
  MergeParams m{};
  m.keys = r.keys;
  m.sums = r.sums;
  m.scores = scores;
  m.finished = finished;
  m.V = vocab;
  m.eos = eos;
  m.K = beams;
  m.select = select;
  m.stretches = sp.stretches;
  m.out_scores = out_scores;
  m.out_rows = out_rows;
  m.out_tokens = out_tokens;
  m.out_finished = out_finished;
  const int row_bytes = sp.stretches * select * (int)sizeof(uint64_t);  // at most 16 KB
  m.rows_per_pass = std::min(beams, kMergeSmem / row_bytes);
  const int smem = m.rows_per_pass * row_bytes;
  static bool attr_done[64] = {false};
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    if (cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMergeSmem) != cudaSuccess)
      return LKV_ERR_CUDA;
    attr_done[dev] = true;
  }
  return launch_pdl(beam_merge_kernel, dim3((unsigned)batch), dim3(kMergeThreads), (size_t)smem, stream, m) ==
                 cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

}  // namespace lkv
