// Beam search's selection over beams and vocabulary (sm_100a).
//
// For batch item b with K beams, scores c[k] and rows of logits x[k][V]:
//     total[k][v] = c[k] + x[k][v] - log sum_u exp x[k][u]
// and the `select` largest totals of the K * V, largest first, equal ones in the order of k * V + v.
// A finished beam has one candidate, its end token at its score.  Totals are compared in 64 bits.
// Within a beam they are ordered as its logits are, so one pass over the logits in their own type
// finds each row's `select` largest together with its maximum and sum of exponentials (fp32):
//
//   beam_rows    A CTA takes a stretch of a row in tiles of 4096 or 8192 values, 16 or 32 in
//                each thread's registers.  It keeps the stretch's best `select` as sorted 64-bit keys (the value as
//                an ordered integer, then the complement of the index, so that no two are equal) and
//                collects the values above the last of them: later tiles mostly hold none, so that a
//                comparison per value is what selection costs.  A tile with too many (the first one)
//                first finds a bar that at least `select` of its values reach: the select-th largest of a
//                warp's 32 lane maxima, in the warp where that is largest, or the (select / 8)-th, in the
//                warp where it is least.  Of values equal to the bar, where they are too many (a masked
//                vocabulary), the first ones are taken; if still too many lie above it, the tile's best are
//                taken out one by one.
//   beam_merge   A CTA per batch item joins each row's stretches two by two, then the rows: lists are
//                sorted, so a candidate's rank is its place in its own list and a binary search in the other.
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
// Values per thread and tile: 32 (tiles of 8192), or 16 where that leaves SMs without a tile.  4 rows of 128256:
// 12.2 us with 32, 10.4 with 16.
constexpr int kPerMany = 32, kPerFew = 16;
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

// The lanes' values sorted from the largest: lane r has the r-th (bitonic).
__device__ __forceinline__ uint32_t warp_sort(uint32_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, v, j);
      const bool larger = ((lane & k) == 0) == ((lane & j) == 0);  // the place that keeps the larger one
      v = larger ? max(v, other) : min(v, other);
    }
  return v;
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

template <typename T, int kPer>
__global__ void __launch_bounds__(kThreads, 3) beam_rows_kernel(const RowsParams p) {
  constexpr int kTile = kThreads * kPer;
  constexpr int VE = 16 / sizeof(T);  // values per 16-byte load
  __shared__ uint64_t cand[kCandidates + kMaxSelect];
  __shared__ uint64_t best[2][kMaxSelect];
  __shared__ uint64_t warp_key[kWarps];
  __shared__ float warp_bar[kWarps], warp_eighth[kWarps];
  __shared__ float2 warp_sum[kWarps];
  __shared__ int counts[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.y;
  const int n = p.select;
  const int64_t out = row * p.stretches + blockIdx.x;
  if (p.finished && p.finished[row]) {
    // one candidate of total 0 + score; behind it the first tokens, at -inf
    if (tid < n) {
      const uint32_t eos = (uint32_t)p.eos, low = ordered(-INFINITY);
      const uint32_t i = tid == 0 ? eos : (uint32_t)(tid - 1) + ((uint32_t)(tid - 1) >= eos ? 1u : 0u);
      p.keys[out * n + tid] =
          blockIdx.x == 0 ? (uint64_t)(tid == 0 ? ordered(0.f) : low) << 32 | (0xffffffffu - i) : 0;
    }
    if (tid == 0) p.sums[out] = make_float2(0.f, 1.f);
    return;
  }
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  // tiles start at 16-byte boundaries, so a row's first may begin before it
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int64_t first = (int64_t)blockIdx.x * p.tiles_per;
  int cur = 0;
  if (tid < n) best[0][tid] = 0;
  if (tid < 2) counts[tid] = 0;
  __syncthreads();
  float m = -INFINITY, sum = 0.f;
  for (int64_t t = first; t < first + p.tiles_per; ++t) {
    const int64_t base = t * kTile - lead;
    if (base >= p.V) break;
    float v[kPer];
    // the index of v[e]: base + (e / VE * kThreads + tid) * VE + e % VE
    auto place = [&](int e) { return (e / VE * kThreads + tid) * VE + e % VE; };
    const bool whole = base >= 0 && base + kTile <= p.V;
    if (whole) {
      const uint4* at = reinterpret_cast<const uint4*>(x + base) + tid;
      uint4 w[kPer / VE];
#pragma unroll
      for (int i = 0; i < kPer / VE; ++i) w[i] = __ldcs(at + i * kThreads);
#pragma unroll
      for (int i = 0; i < kPer / VE; ++i) {
        const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if constexpr (sizeof(T) == 2) v[i * VE + e] = e & 1 ? bf16_hi(u[e / 2]) : bf16_lo(u[e / 2]);
          else v[i * VE + e] = __uint_as_float(u[e]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer / VE; ++i) {
        const int64_t at = base + place(i * VE);
        if (at >= 0 && at + VE <= p.V) {
          const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x + at));
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            if constexpr (sizeof(T) == 2) v[i * VE + e] = e & 1 ? bf16_hi(u[e / 2]) : bf16_lo(u[e / 2]);
            else v[i * VE + e] = __uint_as_float(u[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) v[i * VE + e] = at + e >= 0 && at + e < p.V ? (float)x[at + e] : -INFINITY;
        }
      }
    }
    // the thread's maximum and sum, over all its tiles; a NaN stays in the sum
    float top = v[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) top = fmaxf(top, v[e]);
    const float nm = fmaxf(m, top);
    if (nm != -INFINITY) {
      if (nm != m) sum *= exp2f((m - nm) * kLog2e);
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kPer; ++e) part[e & 3] += ex2_approx((v[e] - nm) * kLog2e);
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      m = nm;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum = v[e] == v[e] ? sum : NAN;
    }
    auto key = [&](int e) -> uint64_t {  // 0 outside the row (below its start the index wraps around)
      const uint32_t i = (uint32_t)base + (uint32_t)place(e);
      return i < (uint32_t)p.V ? (uint64_t)ordered(v[e]) << 32 | ~i : 0;
    };
    // Values above the list's last: an equal one, of a later index, comes behind it.  (A NaN, which counts as
    // -inf, is not below anything; its key tells.)
    const uint64_t last = best[cur][n - 1];
    const bool empty = last == 0;
    const float list_bar = empty ? -INFINITY : from_ordered((uint32_t)(last >> 32));
    const bool some = empty || top > list_bar;
    if (!__syncthreads_or(some)) continue;
    float bar = list_bar;
    bool equal = false;  // whether values equal to the bar count
    // A bar that at least n of the tile's values reach.
    auto tile_bar = [&] {
      const uint32_t sorted = warp_sort(ordered(top), lane);
      if (lane == n - 1) warp_bar[warp] = from_ordered(sorted);
      if (lane == (n + kWarps - 1) / kWarps - 1) warp_eighth[warp] = from_ordered(sorted);
      __syncthreads();
      float least = warp_eighth[0], most = warp_bar[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        most = fmaxf(most, warp_bar[w]);
        least = fminf(least, warp_eighth[w]);
      }
      return fmaxf(most, least);
    };
    // Collects the values above (or equal to) the bar behind the entries that are there.  (The order does not
    // matter: keys are ranked below.)
    auto collect = [&] {
      uint32_t mask = 0;
      if (!(top < bar)) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) mask |= (uint32_t)(equal ? !(v[e] < bar) : v[e] > bar) << e;
      }
      if (mask) {
        int at = atomicAdd(&counts[0], __popc(mask));
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (mask >> e & 1) {
            if (at < kCandidates) cand[at] = key(e);
            ++at;
          }
      }
      __syncthreads();
      return counts[0];
    };
    if (empty) {
      bar = tile_bar();
      equal = true;
    }
    int total = collect();
    if (total > kCandidates) {
      // too many: count what lies above a bar of the tile's own, and on it
      if (!empty) {
        const float own = tile_bar();
        if (own > list_bar) bar = own, equal = true;
      }
      __syncthreads();  // counts are read
      if (tid < 2) counts[tid] = 0;
      __syncthreads();
      int above = 0, level = 0;
      if (!(top < bar)) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          above += v[e] > bar;
          level += equal && !(v[e] < bar) && !(v[e] > bar);
        }
      }
      above = __reduce_add_sync(0xffffffffu, above);
      level = __reduce_add_sync(0xffffffffu, level);
      if (lane == 0 && above) atomicAdd(&counts[0], above);
      if (lane == 0 && level) atomicAdd(&counts[1], level);
      __syncthreads();
      above = counts[0];
      level = counts[1];
      __syncthreads();
      if (tid < 2) counts[tid] = 0;
      if (above > kCandidates - kMaxSelect) {
        // the tile's best, one after another
        uint64_t before = ~0ull;
        for (int r = 0; r < n; ++r) {
          uint64_t big = 0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const uint64_t k = key(e);
            if (k < before) big = max_key(big, k);
          }
          big = warp_max_key(big);
          if (lane == 0) warp_key[warp] = big;
          __syncthreads();
          big = warp_key[0];
          for (int w = 1; w < kWarps; ++w) big = max_key(big, warp_key[w]);
          if (tid == 0) cand[r] = big;
          before = big;
          __syncthreads();
        }
        total = n;
      } else {
        if (above + level > kCandidates) {
          // the first of the values equal to the bar (a NaN counts as -inf)
          equal = false;
          int64_t after = -1;
          for (int r = 0; r < n; ++r) {
            uint32_t next = 0xffffffffu;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
              const int64_t i = base + place(e);
              const float y = v[e] == v[e] ? v[e] : -INFINITY;
              if (y == bar && i > after && i < p.V) next = min(next, (uint32_t)i);
            }
            next = __reduce_min_sync(0xffffffffu, next);
            if (lane == 0) warp_key[warp] = next;
            __syncthreads();
            for (int w = 0; w < kWarps; ++w) next = min(next, (uint32_t)warp_key[w]);
            if (tid == 0) cand[r] = next == 0xffffffffu ? 0 : (uint64_t)ordered(bar) << 32 | (0xffffffffu - next);
            after = next;
            __syncthreads();
          }
          if (tid == 0) counts[0] = n;
        }
        __syncthreads();
        total = min(collect(), kCandidates);
      }
    }
    // the new list: every entry of the old one and of the collected ones finds its rank among all
    if (tid < n) {
      cand[total + tid] = best[cur][tid];
      best[cur ^ 1][tid] = 0;
    }
    __syncthreads();
    if (tid < 2) counts[tid] = 0;
    const int all = total + n;
    for (int a = tid; a < all; a += kThreads) {
      const uint64_t k = cand[a];
      if (k == 0) continue;
      int rank = 0;
#pragma unroll 4
      for (int b = 0; b < all; ++b) rank += cand[b] > k;
      if (rank < n) best[cur ^ 1][rank] = k;
    }
    __syncthreads();
    cur ^= 1;
  }
  // the stretch's maximum and sum: the warps', then the CTA's, in a fixed order
  auto join = [lane](float2 ms, int lanes) {
    float t = ms.x;
    for (int o = lanes / 2; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
    float y = ms.x == t ? ms.y : ms.y * ex2_approx((ms.x - t) * kLog2e);  // (t = -inf: y is 0, or a NaN)
    for (int o = lanes / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    return make_float2(t, y);
  };
  const float2 mine = join(make_float2(m, sum), 32);
  if (lane == 0) warp_sum[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const float2 all = join(warp_sum[lane % kWarps], kWarps);
    if (lane == 0) p.sums[out] = all;
  }
  if (tid < n) p.keys[out * n + tid] = best[cur][tid];
}

struct MergeParams {
  const uint64_t* keys;
  const float2* sums;
  const float* scores;  // [B, K]
  const uint8_t* finished;
  int64_t V, eos;
  int K, select, stretches;
  int log_n, log_lists;  // select and stretches, rounded up to powers of two
  int rows_per_pass;     // rows whose keys fit in shared memory at once
  float* out_scores;
  int64_t* out_rows;
  int64_t* out_tokens;
  uint8_t* out_finished;
};

// How many of the n keys (a power of two), sorted from the largest, are larger than k.
__device__ __forceinline__ int larger(const uint64_t* list, int n, uint64_t k) {
  int at = 0;
  for (int step = n >> 1; step > 0; step >>= 1)
    if (list[at + step - 1] > k) at += step;
  return at + (list[at] > k);
}

constexpr int kMergeThreads = 512;

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const MergeParams p) {
  // [rows_per_pass][1 << log_lists][1 << log_n], padded with zeros, then as much again for half as many lists
  extern __shared__ uint64_t keys[];
  // A total is (x - top) + norm: the maximum is taken off first, so that rows of values like a type's
  // lowest keep their sums' logarithms and their scores.  norm NaN: every total of the row is -inf.
  __shared__ double tops[kMaxBeams], norm[kMaxBeams];
  __shared__ double total[kMaxBeams * kMaxSelect];
  __shared__ uint32_t token[kMaxBeams * kMaxSelect];
  const int b = blockIdx.x, n = p.select, K = p.K, S = p.stretches, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  auto row_norms = [&] {
    for (int k = tid >> 5; k < K; k += kMergeThreads / 32) {  // a warp per row, two stretches per lane
      const int64_t row = (int64_t)b * K + k;
      const int lane = tid & 31;
      const float2 none = make_float2(-INFINITY, 0.f);
      const float2 a = lane < S ? p.sums[row * S + lane] : none, c = lane + 32 < S ? p.sums[row * S + lane + 32] : none;
      float top = fmaxf(a.x, c.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // a stretch of -inf alone adds 0, or a NaN
      auto part = [top](float2 ms) {
        return ms.x == -INFINITY || ms.x == top ? (double)ms.y : (double)ms.y * (double)expf(ms.x - top);
      };
      double sum = part(a) + part(c);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) {
        const bool done = p.finished && p.finished[row];
        const double score = (double)p.scores[row], rest = done ? 0.0 : log(sum);
        tops[k] = done ? 0.0 : (double)top;
        norm[k] = fabs(score) < INFINITY && fabs(tops[k]) < INFINITY && fabs(rest) < INFINITY ? score - rest : NAN;
      }
    }
  };
  for (int k0 = 0; k0 < K; k0 += p.rows_per_pass) {
    const int rows = min(p.rows_per_pass, K - k0);
    const uint64_t* in = p.keys + ((int64_t)b * K + k0) * S * n;
    const int log_n = p.log_n, pad = 1 << log_n;
    uint64_t* from = keys;
    uint64_t* to = keys + ((int64_t)p.rows_per_pass << (p.log_lists + log_n));
    __syncthreads();
    for (int i = tid; i < rows << (p.log_lists + log_n); i += kMergeThreads) {
      const int at = i & (pad - 1), list = i >> log_n, s = list & ((1 << p.log_lists) - 1), r = list >> p.log_lists;
      from[i] = at < n && s < S ? in[(r * S + s) * n + at] : 0;
    }
    if (k0 == 0) row_norms();
    __syncthreads();
    // lists 2 s and 2 s + 1 become list s, until a row has one
    for (int log_lists = p.log_lists; log_lists > 0; --log_lists) {
      for (int i = tid; i < rows << (log_lists + log_n); i += kMergeThreads) {
        const int list = i >> log_n;
        const uint64_t k = from[i];
        const int rank = (i & (pad - 1)) + larger(from + ((list ^ 1) << log_n), pad, k);
        // (zeros, past a list's end, come behind both lists' others, some of them to the same places)
        if (rank < pad) to[((list >> 1) << log_n) + rank] = k;
      }
      __syncthreads();
      uint64_t* t = from;
      from = to;
      to = t;
    }
    for (int i = tid; i < rows * n; i += kMergeThreads) {
      const int r = i / n, rank = i - r * n;
      const uint64_t k = from[(r << log_n) + rank];
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
  bool few;
};
// About two CTAs per SM over all rows, whole tiles each: a stretch's first tile costs as much as four others.
Split split_rows(int64_t rows, int64_t V, int sms) {
  const int64_t large = kThreads * kPerMany, small = kThreads * kPerFew;
  const bool few = rows * ((V + 7 + large - 1) / large) <= sms;
  const int64_t tile = few ? small : large, tiles = (V + 7 + tile - 1) / tile;
  const int64_t s = std::min<int64_t>({tiles, (int64_t)kMaxStretches, std::max<int64_t>(1, 2ll * sms / rows)});
  const int64_t per = (tiles + s - 1) / s;
  return {(int)((tiles + per - 1) / per), (int)per, few};
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
  const auto kern = fp32 ? (sp.few ? beam_rows_kernel<float, kPerFew> : beam_rows_kernel<float, kPerMany>)
                         : (sp.few ? beam_rows_kernel<__nv_bfloat16, kPerFew> : beam_rows_kernel<__nv_bfloat16, kPerMany>);
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
  while (1 << m.log_n < select) ++m.log_n;
  while (1 << m.log_lists < sp.stretches) ++m.log_lists;
  const int row_bytes = (3 << (m.log_n + m.log_lists)) / 2 * (int)sizeof(uint64_t) + (int)sizeof(uint64_t);  // 24 KB at most
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
