// Beam search's selection over beams and vocabulary (sm_100a).
//
// For batch item b with K beams, scores c[k] and rows of logits x[k][V]:
//     total[k][v] = c[k] + x[k][v] - log sum_u exp x[k][u]
// and the `select` largest totals of the K * V, largest first, equal ones in the order of k * V + v.
// A finished beam has one candidate, its end token at its score.  Totals are compared in 64 bits.
// Within a beam they are ordered as its logits are, so one pass over the logits in their own type
// finds each row's `select` largest together with its maximum and sum of exponentials (fp32):
//
//   beam_rows    A CTA takes a stretch of a row; its warps take pieces of 32 x 16 bytes by turns, each for
//                itself.  A warp keeps its best 32 as sorted 64-bit keys, one per lane (the value as an
//                ordered integer, then the complement of the index, so that no two are equal), and puts the
//                few values that may be among the stretch's best into their places one by one; for the rest
//                selection costs a comparison of a lane's maximum.  What they are held against is a bar
//                that at least `select` values of the stretch reach: the select-th largest of the four best
//                of every warp, which the warps leave in shared memory as they rise, at first by their
//                lanes' maxima.  (How old those are that a warp finds does not change the result, only how
//                many values it looks at.)
//                At the end the warps' lists are merged two by two (bitonic).
//   beam_merge   A CTA per batch item joins each row's stretches two by two, then the rows: lists are
//                sorted, so a candidate's rank is its place in its own list and a binary search in the other.
//
// Bound by HBM for many rows and by the latencies of two launches, a CTA's few steps over its stretch and the join's
// rounds for few: 4 rows of 128256 bf16 logits take 8.7 us, 128 rows of 50001 in fp32 (25.6 MB) 22, 512 of
// 32000 in bf16 (32.8 MB) 25.

#include <math.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace lkv {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kGroupValues = 16;  // a lane's values that are loaded together, one group ahead
constexpr int kMaxSelect = 32;
constexpr int kMaxBeams = 64;
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

// The 32 largest of two sorted lists, one key of each per lane, sorted: the second is given reversed, so that the
// larger of each lane's pair are the 32 largest and form a bitonic sequence.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, uint64_t b_reversed, int lane) {
  uint64_t v = max_key(a, b_reversed);
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, v, j);
    v = (lane & j) == 0 ? max_key(v, other) : (v < other ? v : other);
  }
  return v;
}

struct RowsParams {
  const void* logits;
  int64_t row_stride;
  int64_t V;
  const uint8_t* finished;  // [rows] or null
  int64_t eos;
  int select, stretches;
  int pieces_per;  // of a stretch: kWarps x 32 x 16 bytes each
  uint64_t* keys;  // [rows][stretches][select], sorted, 0 past the last
  float2* sums;    // [rows][stretches]: maximum, sum of exp(x - maximum)
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) beam_rows_kernel(const RowsParams p) {
  constexpr int VE = 16 / sizeof(T);  // values of a lane's 16 bytes
  constexpr int kGroup = kGroupValues / VE;
  __shared__ uint64_t lists[kWarps][32];
  __shared__ float2 warp_sum[kWarps];
  __shared__ volatile uint32_t known[kWarps * 4];  // ordered values: each warp's best four so far, at least
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.y;
  const int n = p.select;
  const int64_t out = row * p.stretches + blockIdx.x;
  if (p.finished && p.finished[row]) {
    // one candidate of total 0 + score; behind it the first tokens, at -inf
    const int i = threadIdx.x;
    if (i < n) {
      const uint32_t eos = (uint32_t)p.eos, low = ordered(-INFINITY);
      const uint32_t token = i == 0 ? eos : (uint32_t)(i - 1) + ((uint32_t)(i - 1) >= eos ? 1u : 0u);
      p.keys[out * n + i] = blockIdx.x == 0 ? (uint64_t)(i == 0 ? ordered(0.f) : low) << 32 | ~token : 0;
    }
    if (i == 0) p.sums[out] = make_float2(0.f, 1.f);
    return;
  }
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  // pieces start at 16-byte boundaries, so a row's first may begin before it
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  // piece j of this warp: 32 lanes x VE values from index first + j * kWarps * 32 * VE on
  constexpr uint32_t kStep = kWarps * 32 * VE;
  const int64_t first = ((int64_t)blockIdx.x * p.pieces_per * kWarps + warp) * (32 * VE) + lane * VE - lead;
  // a lane's 16 bytes lie in the row where its first index, in 32 bits, is below this (one below the row's start wraps)
  const uint32_t inside = p.V >= VE ? (uint32_t)(p.V - VE) + 1 : 0;
  auto load = [&](uint4 (&w)[kGroup], int j0) {  // returns which pieces are there
    uint32_t there = 0;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      const uint32_t i = (uint32_t)first + (uint32_t)(j0 + j) * kStep;
      if (j0 + j < p.pieces_per && i < inside) {
        w[j] = __ldcs(reinterpret_cast<const uint4*>(x + i));
        there |= 1u << j;
      }
    }
    return there;
  };
  float m = -INFINITY, sum = 0.f;  // this lane's
  uint64_t list = 0, last = 0;     // lane r: the warp's r-th best key; the select-th
  float bar = -INFINITY;           // what may be among the stretch's best is above it
  bool all = true;                 // not even that is known: fewer than select values so far
  // A bar from what the warps have left in shared memory and this one's own list.  Values equal to another warp's
  // may come before them: that bar is the next value below.
  static_assert(kWarps * 4 == 32, "one of the known values for each lane");
  auto raise = [&] {
    uint32_t below = max(__shfl_sync(0xffffffffu, warp_sort(known[lane], lane), n - 1), 1u) - 1;
    if (below == 0x7fffffffu) --below;  // -0, which is no less than 0
    const uint32_t at = max(below, (uint32_t)(last >> 32));
    all = at < ordered(-INFINITY);
    bar = all ? -INFINITY : from_ordered(at);
  };
  uint4 w[kGroup];
  uint32_t there = load(w, 0);
  for (int j0 = 0; j0 < p.pieces_per; j0 += kGroup) {
    if (j0 && first - lane * VE + (int64_t)j0 * kStep >= p.V) break;  // the same for the warp
    float v[kGroup][VE], tops[kGroup];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      if (there >> j & 1) {
        const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if constexpr (sizeof(T) == 2) v[j][e] = e & 1 ? bf16_hi(u[e / 2]) : bf16_lo(u[e / 2]);
          else v[j][e] = __uint_as_float(u[e]);
        }
      } else {
        const uint32_t i = (uint32_t)first + (uint32_t)(j0 + j) * kStep;
#pragma unroll
        for (int e = 0; e < VE; ++e)
          v[j][e] = j0 + j < p.pieces_per && i + e < (uint32_t)p.V ? (float)x[i + e] : -INFINITY;
      }
      tops[j] = v[j][0];
#pragma unroll
      for (int e = 1; e < VE; ++e) tops[j] = fmaxf(tops[j], v[j][e]);
      top = fmaxf(top, tops[j]);
    }
    there = load(w, j0 + kGroup);
    // maximum and sum; a NaN stays in the sum
    const float nm = fmaxf(m, top);
    if (nm != -INFINITY) {
      if (nm != m) sum *= ex2_approx((m - nm) * kLog2e);
      m = nm;
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < VE; ++e) part += ex2_approx((v[j][e] - nm) * kLog2e);
        sum += part;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
#pragma unroll
        for (int e = 0; e < VE; ++e) sum = v[j][e] == v[j][e] ? sum : NAN;
    }
    // the warp's best
    if (j0 == 0) {
      const uint32_t sorted = warp_sort(ordered(top), lane);
      if (lane < 4) known[warp * 4 + lane] = sorted;
      asm volatile("bar.sync 1, %0;" ::"n"(kThreads));
    }
    if (!__any_sync(0xffffffffu, all || top > bar)) continue;
    raise();
    if (!__any_sync(0xffffffffu, all || top > bar)) continue;
    bool changed = false;
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      if (!__any_sync(0xffffffffu, all || tops[j] > bar)) continue;
      const uint32_t i0 = (uint32_t)first + (uint32_t)(j0 + j) * kStep;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float y = v[j][e];
        if (!__any_sync(0xffffffffu, all || y > bar)) continue;
        const uint32_t i = i0 + e;
        const bool valid = (all || y > bar) && i < (uint32_t)p.V && j0 + j < p.pieces_per;
        const uint64_t key = valid ? (uint64_t)ordered(y) << 32 | ~i : 0;
        uint32_t who = __ballot_sync(0xffffffffu, key > last);
        changed |= who != 0;
        while (who) {
          const uint64_t k = __shfl_sync(0xffffffffu, key, __ffs(who) - 1);
          const int place = __popc(__ballot_sync(0xffffffffu, list > k));
          const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
          list = lane < place ? list : lane == place ? k : up;
          last = __shfl_sync(0xffffffffu, list, n - 1);
          who &= who - 1;
          who &= __ballot_sync(0xffffffffu, key > last);
        }
      }
    }
    if (changed) {
      if (lane < 4) known[warp * 4 + lane] = max(known[warp * 4 + lane], (uint32_t)(list >> 32));
    }
  }
  // the stretch's list, maximum and sum: the warps', then the CTA's, in a fixed order
  auto join = [lane](float2 ms, int lanes) {
    float t = ms.x;
    for (int o = lanes / 2; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
    float y = ms.x == t ? ms.y : ms.y * ex2_approx((ms.x - t) * kLog2e);  // (t = -inf: y is 0, or a NaN)
    for (int o = lanes / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    return make_float2(t, y);
  };
  const float2 mine = join(make_float2(m, sum), 32);
  if (lane == 0) warp_sum[warp] = mine;
#pragma unroll
  for (int half = kWarps / 2; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) lists[warp][lane] = list;
    __syncthreads();
    if (warp < half) list = merge_lists(list, lists[warp + half][31 - lane], lane);
  }
  if (warp == 0) {
    const float2 all = join(warp_sum[lane % kWarps], kWarps);
    if (lane == 0) p.sums[out] = all;
    if (lane < n) p.keys[out * n + lane] = list;
  }
}

struct MergeParams {
  const uint64_t* keys;
  const float2* sums;
  const float* scores;  // [B, K]
  const uint8_t* finished;
  int64_t V, eos;
  int K, select, stretches;
  int log_n, log_lists, log_beams;  // select, stretches and beams, rounded up to powers of two
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

// A total as an integer of the same order, above 0.
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double from_ordered(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

constexpr int kMergeThreads = 512;

// Lists of 1 << log_n entries, sorted from the largest, two by two into half as many, until there is one for
// each 1 << log_lists; of equal entries the earlier list's come first (k + 1 in its place in the search).  Where a
// payload goes with the keys it moves along.  Returns with `from` the result's place.
template <bool PAYLOAD>
__device__ __forceinline__ void merge_rounds(uint64_t*& from, uint64_t*& to, uint32_t*& pay, uint32_t*& pay_to, int groups,
                                             int log_lists, int log_n) {
  const int pad = 1 << log_n;
  for (; log_lists > 0; --log_lists) {
    for (int i = threadIdx.x; i < groups << (log_lists + log_n); i += kMergeThreads) {
      const int list = i >> log_n;
      const uint64_t k = from[i];
      // an equal entry of the list before comes first: it counts as larger
      const int rank = (i & (pad - 1)) + larger(from + ((list ^ 1) << log_n), pad, PAYLOAD && (list & 1) && k ? k - 1 : k);
      // (zeros, past a list's end, come behind both lists' others, some of them to the same places)
      if (rank < pad) {
        to[((list >> 1) << log_n) + rank] = k;
        if (PAYLOAD) pay_to[((list >> 1) << log_n) + rank] = pay[i];
      }
    }
    __syncthreads();
    uint64_t* t = from;
    from = to;
    to = t;
    if (PAYLOAD) {
      uint32_t* u = pay;
      pay = pay_to;
      pay_to = u;
    }
  }
}

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const MergeParams p) {
  // [K][1 << log_lists][1 << log_n], padded with zeros, then as much again for half as many lists
  extern __shared__ uint64_t keys[];
  // A total is (x - top) + norm: the maximum is taken off first, so that rows of values like a type's
  // lowest keep their sums' logarithms and their scores.  norm NaN: every total of the row is -inf.
  __shared__ double tops[kMaxBeams], norm[kMaxBeams];
  __shared__ uint64_t total[kMaxBeams * kMaxSelect * 3 / 2];  // ordered totals: a list of 1 << log_n for each beam
  __shared__ uint32_t from_where[kMaxBeams * kMaxSelect * 3 / 2];  // the beam and the place in its list
  __shared__ uint32_t token[kMaxBeams * kMaxSelect];
  __shared__ bool ended[kMaxBeams];  // read before anything is written: the outputs may be the inputs' buffers
  const int b = blockIdx.x, n = p.select, K = p.K, S = p.stretches, tid = threadIdx.x;
  const int log_n = p.log_n, pad = 1 << log_n;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = tid & 31;
  const float2 none = make_float2(-INFINITY, 0.f);
  auto sums_at = [&](int k, int s) { return k < K && s < S ? __ldcg(p.sums + ((int64_t)b * K + k) * S + s) : none; };
  float2 a = sums_at(tid >> 5, lane), c = sums_at(tid >> 5, lane + 32);  // a warp per row, two stretches per lane
  for (int i = tid; i < 1 << (p.log_beams + log_n); i += kMergeThreads) total[i] = 0;
  const int entries = K << (p.log_lists + log_n);
  const uint64_t* in = p.keys + (int64_t)b * K * S * n;
  uint64_t* lists = keys;
  uint64_t* lists_to = keys + entries;
  uint32_t* unused = nullptr;
  for (int i0 = tid; i0 < entries; i0 += 8 * kMergeThreads) {  // eight loads in flight
    uint64_t k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * kMergeThreads;
      const int at = i & (pad - 1), list = i >> log_n, s = list & ((1 << p.log_lists) - 1), r = list >> p.log_lists;
      const bool there = i < entries && at < n && s < S;
      k[j] = __ldcg(in + (there ? (r * S + s) * n + at : 0));
      if (!there) k[j] = 0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + j * kMergeThreads < entries) lists[i0 + j * kMergeThreads] = k[j];
  }
  for (int k = tid >> 5; k < K; k += kMergeThreads / 32) {
    const int64_t row = (int64_t)b * K + k;
    float top = fmaxf(a.x, c.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // a stretch of -inf alone adds 0, or a NaN
    auto part = [top](float2 ms) {
      return ms.x == -INFINITY || ms.x == top ? (double)ms.y : (double)(ms.y * ex2_approx((ms.x - top) * kLog2e));
    };
    double sum = part(a) + part(c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      const bool done = p.finished && p.finished[row];
      // log(f 2^e) = e log 2 + log f with f in 1 .. 2, whose logarithm fp32 has to 2^-24
      const int e = ilogb(sum);
      const double score = (double)p.scores[row];
      const double rest = done ? 0.0 : e * 0.6931471805599453 + (double)logf((float)scalbn(sum, -e));
      ended[k] = done;
      tops[k] = done ? 0.0 : (double)top;
      norm[k] = fabs(score) < INFINITY && fabs(tops[k]) < INFINITY && fabs(rest) < INFINITY ? score - rest : NAN;
    }
    a = sums_at(k + kMergeThreads / 32, lane);
    c = sums_at(k + kMergeThreads / 32, lane + 32);
  }
  __syncthreads();
  merge_rounds<false>(lists, lists_to, unused, unused, K, p.log_lists, log_n);
  for (int i = tid; i < K << log_n; i += kMergeThreads) {
    const int k = i >> log_n, rank = i & (pad - 1);
    if (rank >= n) continue;
    const uint64_t key = lists[i];
    const double t = ((double)from_ordered((uint32_t)(key >> 32)) - tops[k]) + norm[k];
    const bool alive = norm[k] == norm[k];
    // all totals of a row without a finite score or sum are -inf: its first tokens, in their order
    total[i] = ordered(alive && t == t ? t : -INFINITY);
    from_where[i] = (uint32_t)i;
    token[k * n + rank] = alive ? 0xffffffffu - (uint32_t)key : (uint32_t)rank;
  }
  __syncthreads();
  uint64_t* from = total;
  uint64_t* to = total + (1 << (p.log_beams + log_n));
  uint32_t* pay = from_where;
  uint32_t* pay_to = from_where + (1 << (p.log_beams + log_n));
  merge_rounds<true>(from, to, pay, pay_to, 1, p.log_beams, log_n);
  if (tid < n) {
    const int k = (int)(pay[tid] >> log_n);
    const uint32_t v = token[k * n + (pay[tid] & (pad - 1))];
    const int64_t row = (int64_t)b * K + k, at = (int64_t)b * n + tid;
    p.out_scores[at] = (float)from_ordered(from[tid]);
    p.out_rows[at] = row;
    p.out_tokens[at] = v;
    if (p.out_finished) p.out_finished[at] = (int64_t)v == p.eos || ended[k];
  }
}

struct Split {
  int stretches, pieces;
};
constexpr int kMergeSmem = 128 * 1024;
// What the join holds of a row: `lists` lists of 1 << log_n keys, and half as many of the next round.
int64_t join_bytes(int64_t lists, int log_n) { return ((3 * lists << log_n) / 2 + 1) * (int64_t)sizeof(uint64_t); }

// Stretches for four CTAs per SM over all rows, all at once (16 items of 8 beams over 50001 tokens: 22.0 us, with
// three 23.6, with six 25.8), of two pieces for each warp at least, and no more than the join can hold of
// all beams at once (16 beams over 200000 tokens, the 32 best:
// 33 us; in several passes 42 to 66).
Split split_rows(int64_t rows, int beams, int log_n, int64_t V, int elem, int sms) {
  const int64_t piece = kThreads * 16 / elem, pieces = (V + 16 / elem - 1 + piece - 1) / piece;
  int64_t most = kMaxStretches;
  while (most > 1 && beams * join_bytes(most, log_n) > kMergeSmem) most /= 2;
  const int64_t s = std::min<int64_t>({(pieces + 1) / 2, most, std::max<int64_t>(1, 4ll * sms / rows)});
  const int64_t per = (pieces + s - 1) / s;
  return {(int)((pieces + per - 1) / per), (int)per};
}

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
  MergeParams m{};
  while (1 << m.log_n < select) ++m.log_n;
  const Split sp = split_rows(rows, beams, m.log_n, vocab, fp32 ? 4 : 2, sms);
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
  r.pieces_per = sp.pieces;
  r.sums = static_cast<float2*>(workspace);
  r.keys = reinterpret_cast<uint64_t*>(r.sums + entries);
  const dim3 grid((unsigned)sp.stretches, (unsigned)rows);
  const auto kern = fp32 ? beam_rows_kernel<float> : beam_rows_kernel<__nv_bfloat16>;
  if (launch_pdl(kern, grid, dim3(kThreads), 0, stream, r) != cudaSuccess) return LKV_ERR_CUDA;
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
  while (1 << m.log_lists < sp.stretches) ++m.log_lists;
  while (1 << m.log_beams < beams) ++m.log_beams;
  const int64_t smem = beams * join_bytes(1ll << m.log_lists, m.log_n);  // kMergeSmem at most (split_rows)
  static std::atomic<bool> attr_done[64];
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
