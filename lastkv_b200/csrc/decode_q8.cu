// Split-KV decode over a cache whose older pages are held in 8 bits (sm_100a).
//
// Row b attends to seq_k[b] keys: its first num_q8[b] block-table columns are 8-bit pages
// (pages_q8.cuh), the rest pages of the bf16 pool.  Per KV head, with the GQA group's query heads
// folded into one tile of 8 columns,
//     S^T[16 keys, 8 heads] = K[16, D] Q^T          (mma m16n8k16, fp32 sums)
//     s = S * key scale * softmax scale,  online softmax in fp32
//     O^T[D, 8 heads] += V^T[D, 16] (p * value scale)^T
// The scales belong to 8 tokens, the rows of an accumulator, and never touch the codes.  The codes
// are whole numbers up to 127 and enter the products as f16, exactly: a byte q + 128 becomes 1024 +
// 128 + q by one byte permutation that puts it under f16's exponent byte, and one subtraction
// takes the 1152 off (bf16, with 7 bits of mantissa, took 3.5 instructions for two codes instead of 2).
// - Q: a row's heads are divided by a power of two that brings their largest value to 1 .. 2 and rounded to
//   f16: exact but for values below 2^-17 of the largest, which are rounded at 2^-25 of it.
// - p * value scale: with t = s + log2(value scale) and M its running maximum, the product is 2^(t - M),
//   in 0 .. 1; times 2^15 it uses f16's whole range, 11 bits down to
//   2^-29 of the largest and 2^-40 of it as the smallest step.  A token's part of the sum of weights is that
//   number (in fp32) divided by the value scale; the scales of a row may lie 2^90 apart (zero aside), further the
//   number flushes to 0 for tokens that still count.
// bf16 pages keep bf16 operands, and the same M with a value scale of 1 (a slot has pages of one kind, and a row's
// 8-bit ones come first: their products are in the fp32 sums before a larger M).
//
// Bound by HBM: an 8-bit page is half a bf16 page's bytes.  Work is counted in slots of equal bytes, one bf16
// page or two 8-bit pages of one KV head.  The rows' slots lie end to end, (row, head) after
// (row, head), each behind the places of what a (row, head) costs by itself, and every CTA takes the same number
// of places, so ragged rows cost no balance; a (row, head)'s part within a CTA is a piece, whose normalised partial goes to the workspace, and
// join_pieces_kernel joins each row's pieces.  Per CTA one warp fills a ring of slots (an 8-bit page's codes by
// a bulk copy and its scales by cp.async, a bf16 page's halves by TMA), 6 warps take the slots in turn.

#include <math.h>

#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <mutex>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"
#include "pages_q8.cuh"

namespace lkv {

namespace {

struct DecodeQ8Params {
  const __nv_bfloat16* q;
  int64_t q_stride_tok;
  const uint8_t* codes;
  const float* scales;
  int64_t q8_pages;
  int64_t pool_pages;  // 0: no bf16 pool
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* num_q8;  // or null: every column
  const int32_t* seq_k;
  __nv_bfloat16* out;
  int64_t out_stride_tok;
  float* lse;              // natural log [B, Hq] or null
  const float* out_scale;  // [Hq] or null
  float* part_o;           // [pieces][GROUP][D], normalised
  float* part_lse;         // [pieces][GROUP], natural log
  int* first_place;        // [B + 1]: the rows' first places and the places per CTA, written for join_pieces_kernel
  int* err;
  int B, Hq, Hkv, W;
  int whole;  // 1: CTAs take whole (row, head)s and write the result themselves
  float scale_log2;
  int keep_pages;  // leading columns that stay in L2
};

constexpr int kNW = 6;  // consumer warps: with the producer 14 warps on an SM, 128 registers for a thread
constexpr int kThreads = (kNW + 1) * 32;
constexpr int kLeastSlots = kNW;  // of a CTA that has any: a slot for each warp

template <int D>
struct Q8Cfg {
  // 96 KB of slots: two CTAs per SM.  A multiple of the warps, so that a ring place is always the same warp's: two
  // warps could wait for two different copies into one place with the same barrier parity.
  static constexpr int RING = D == 128 ? 12 : 24;
  static_assert(RING % kNW == 0, "a ring place belongs to one warp");
  // Slots that the producer waits for and copies at once, a lane per half: one after another they took it
  // 600 cycles each, more than a slot's time at the memory's rate.
  static constexpr int BATCH = RING / 3;
  static constexpr int HALVES = D / 64;
  static constexpr int TILE_BYTES = kPageTokens * 128;    // 16 rows x 64 bf16
  static constexpr int CODE_BYTES = 2 * kPageTokens * D;  // keys and values of an 8-bit page
  static constexpr int SLOT_BYTES = 2 * CODE_BYTES;       // two 8-bit pages, or one bf16 page
  static constexpr int OSTRIDE = D + 4;
  static constexpr int OFF_SCALE = RING * SLOT_BYTES;     // two pages' scales per slot
  static constexpr int OFF_Q = OFF_SCALE + RING * 32;     // bf16 Q operands of the current piece
  // join area: o [kNW][2 heads][OSTRIDE], then m and l [kNW][8]
  static constexpr int OFF_JOIN = OFF_Q + (D / 16) * 32 * 8;
  static constexpr int OFF_BAR = OFF_JOIN + kNW * 2 * OSTRIDE * 4 + 2 * kNW * 8 * 4;
  static constexpr int SMEM_BYTES = 1024 + OFF_BAR + 2 * RING * 8 + 64;
};

__device__ __forceinline__ float max_over_rows(float v) {  // over the 8 lanes that share lane & 3
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

__device__ __forceinline__ float sum_over_rows(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// D = A(16x16, row) * B(16x8, col) + D, f16 inputs, fp32 accumulate.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes to shared memory, and this thread's arrival on a barrier once its copies so far are there.
__device__ __forceinline__ void async_copy16(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void async_copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

constexpr float kWeightLog2 = 15.f;  // weights of the products are times 2^15

// The slots of row b.
struct Row {
  int n, npages, nh, hs, slots;  // keys, pages, 8-bit pages, their slots, all slots of a head
};
__device__ __forceinline__ Row row_of(const DecodeQ8Params& p, int b) {
  Row r;
  r.n = max(0, p.seq_k[b]);
  r.npages = min((int)(((int64_t)r.n + kPageTokens - 1) / kPageTokens), p.W);
  r.n = min(r.n, r.npages * kPageTokens);
  r.nh = p.num_q8 ? min(max(p.num_q8[b], 0), r.npages) : r.npages;
  r.hs = (r.nh + 1) / 2;
  r.slots = r.hs + r.npages - r.nh;
  return r;
}

// What a (row, head) costs besides its slots, in slots: its Q, the join of the warps, the partial.
constexpr int kPieceCost = 6;

// A (row, head)'s places in the order that CTAs share: kPieceCost of its own, then one per slot.
__device__ __forceinline__ int places(const Row& r) { return r.slots ? r.slots + kPieceCost : 0; }

// What a CTA takes: `left` places from place `at` of (row b, head hk) on (whole: `left` (row, head)s).
struct Share {
  Row r;  // of row b
  int b, hk, at, piece, left;
};

// A piece: slots [s0, s1) of (row b, head hk).
struct Piece {
  Row r;
  int b, hk, s0, s1, id;
};

// The next piece of a share; false where it ends.  Every warp walks its copy of the share.
__device__ __forceinline__ bool next_piece(const DecodeQ8Params& p, Share& s, Piece& x) {
  if (s.left <= 0) return false;
  if (s.hk == p.Hkv) {
    s.hk = 0;
    do {
      if (++s.b >= p.B) return false;
      s.r = row_of(p, s.b);
      if (s.r.slots == 0 && !p.whole) s.piece += p.Hkv;  // no pieces, but their places among them
    } while (s.r.slots == 0 && !p.whole);
  }
  x.r = s.r;
  x.b = s.b;
  x.hk = s.hk++;
  x.id = s.piece++;
  if (p.whole) {
    x.s0 = 0;
    x.s1 = s.r.slots;
    --s.left;
    return true;
  }
  const int take = min(s.left, s.r.slots + kPieceCost - s.at);
  x.s0 = max(0, s.at - kPieceCost);
  x.s1 = s.at + take - kPieceCost;
  s.left -= take;
  s.at = 0;
  return x.s1 > x.s0;  // a share that ends before a (row, head)'s first slot ends there
}

// The CTA's share, called by all threads.  Piece u of the (row, head)s in order, cut at CTA c's first place, is
// piece u + c.  (All places together are below 2^31: the host checks the tables' size.)
__device__ Share share_of(const DecodeQ8Params& p, int* sm, int* sm_row) {
  Share s{};
  const unsigned cta = blockIdx.x, ctas = gridDim.x;
  if (p.whole) {
    const unsigned units = (unsigned)p.B * p.Hkv;
    const unsigned u0 = (unsigned)((uint64_t)units * cta / ctas), u1 = (unsigned)((uint64_t)units * (cta + 1) / ctas);
    s.b = (int)(u0 / p.Hkv);
    s.hk = (int)(u0 % p.Hkv);
    s.piece = (int)u0;
    s.left = (int)(u1 - u0);
    s.r = row_of(p, s.b);
    return s;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto prefix = [lane](int v) {  // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    return v;
  };
  auto share = [ctas](int all) {
    return max((int)(((unsigned)all + ctas - 1) / ctas), kLeastSlots + kPieceCost);
  };
  int total, per, start;  // start: the first place of the row that holds the CTA's first
  int64_t first;
  if (p.B <= 32) {  // every warp for itself
    Row r{};
    if (lane < p.B) r = row_of(p, lane);
    const int here = places(r) * p.Hkv, upto = prefix(here);
    total = __shfl_sync(0xffffffffu, upto, 31);
    per = share(total);
    first = (int64_t)per * cta;
    if (cta == 0 && warp == 0) {
      if (lane < p.B) p.first_place[lane] = upto - here;
      if (lane == 0) p.first_place[p.B] = per;
    }
    if (first >= total) return s;
    s.b = __ffs(__ballot_sync(0xffffffffu, upto > first)) - 1;
    start = __shfl_sync(0xffffffffu, upto - here, s.b);
    s.r.n = __shfl_sync(0xffffffffu, r.n, s.b);
    s.r.npages = __shfl_sync(0xffffffffu, r.npages, s.b);
    s.r.nh = __shfl_sync(0xffffffffu, r.nh, s.b);
    s.r.hs = (s.r.nh + 1) / 2;
    s.r.slots = s.r.hs + s.r.npages - s.r.nh;
  } else {
    constexpr int WARPS = kThreads / 32;
    int mine = 0;
    for (int b = threadIdx.x; b < p.B; b += kThreads) mine += places(row_of(p, b));
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sm[warp] = mine;
    __syncthreads();
    total = 0;
    for (int w = 0; w < WARPS; ++w) total += sm[w];
    total *= p.Hkv;
    per = share(total);
    first = (int64_t)per * cta;
    if (first >= total && cta != 0) return s;
    // CTA 0 goes through all rows, for join_pieces_kernel
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const int here = b < p.B ? places(row_of(p, b)) * p.Hkv : 0;
      const int upto = prefix(here);
      __syncthreads();  // sm is read
      if (lane == 31) sm[warp] = upto;
      __syncthreads();
      int at = before + upto - here;
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) at += sm[w];
        before += sm[w];
      }
      if (cta == 0 && b < p.B) {
        p.first_place[b] = at;
        if (b == p.B - 1) p.first_place[p.B] = per;
      }
      if (here > 0 && at <= first && first < at + here) {
        *sm_row = b;
        sm[WARPS] = at;
      }
      if (cta != 0 && before > first) break;  // the same for all threads
    }
    __syncthreads();
    if (first >= total) return s;
    s.b = *sm_row;
    start = sm[WARPS];
    s.r = row_of(p, s.b);
  }
  const unsigned unit = s.r.slots + kPieceCost, off = (unsigned)((int)first - start);
  s.hk = (int)(off / unit);
  s.at = (int)(off % unit);
  s.piece = s.b * p.Hkv + s.hk + (int)cta;
  s.left = min(per, total - (int)first);
  return s;
}

template <int D, int GROUP>
__global__ void __launch_bounds__(kThreads, 2)
    decode_q8_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                     const DecodeQ8Params p) {
  using Cfg = Q8Cfg<D>;
  constexpr int RING = Cfg::RING, KT = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* jo = reinterpret_cast<float*>(smem + Cfg::OFF_JOIN);
  float* jm = jo + kNW * 2 * Cfg::OSTRIDE;
  float* jl = jm + kNW * 8;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* empty = full + RING;
  volatile int* fail_flag = reinterpret_cast<volatile int*>(empty + RING);
  __shared__ int sm_sum[kThreads / 32 + 1];
  __shared__ int sm_row;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < RING; ++s) {
      mbar_init(&full[s], 3);  // the expected bytes, and the scales of both halves
      mbar_init(&empty[s], 1);
    }
    *fail_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  Share share = share_of(p, sm_sum, &sm_row);
  Piece x;
  uint32_t gs = 0;  // slots of this CTA's earlier pieces: slot k of a piece has ring place (gs + k) % RING

  if (warp == kNW) {
    // ------------------------------------------------------------ producer
    // Lane 2 i + u copies half u of the i-th slot of a group of 16: an 8-bit page (its codes and scales), or the
    // keys (u = 0) or values (u = 1) of a bf16 page.
    if (p.pool_pages && lane == 0) {
      tma_prefetch_desc(&tmk);
      tma_prefetch_desc(&tmv);
    }
    const uint64_t pol_first = policy_evict_first(), pol_last = policy_evict_last();
    const int u = lane & 1;
    bool ok = true;
    while (ok && next_piece(p, share, x)) {
      const int32_t* row = p.bt + (int64_t)x.b * p.bt_stride;
      const int count = x.s1 - x.s0;
      // this lane's block-table column of the group from slot k on (-1: none), and its page, read a group ahead
      auto column = [&](int k) {
        const int sl = x.s0 + k + (lane >> 1);
        if (sl >= x.s1) return -1;
        if (sl >= x.r.hs) return x.r.nh + sl - x.r.hs;
        return 2 * sl + u < x.r.nh ? 2 * sl + u : -1;
      };
      int col = column(0);
      int id = col >= 0 ? __ldg(row + col) : 0;
      for (int k0 = 0; ok && k0 < count; k0 += 16) {
        const int c = col, pid = id;
        col = column(k0 + 16);
        if (col >= 0) id = __ldg(row + col);
        const bool q8 = c >= 0 && c < x.r.nh;
        const bool bad = c >= 0 && (pid < 0 || (int64_t)pid >= (q8 ? p.q8_pages : p.pool_pages));
        const uint32_t bytes = c >= 0 && !bad ? Cfg::CODE_BYTES : 0;
        const uint32_t both = bytes + __shfl_xor_sync(0xffffffffu, bytes, 1);
        const uint64_t pol = c < p.keep_pages ? pol_last : pol_first;
        const int64_t block = (int64_t)pid * p.Hkv + x.hk;
        for (int i0 = 0; i0 < min(16, count - k0); i0 += Cfg::BATCH) {
          const int i = (lane >> 1) - i0;
          const bool mine = i >= 0 && i < Cfg::BATCH && k0 + i0 + i < count;
          const uint32_t at = gs + max(i, 0);
          const int s = (int)(at % RING);
          ok = __all_sync(0xffffffffu, !mine || mbar_wait(&empty[s], ((at / RING) & 1u) ^ 1u));
          if (!ok) break;
          uint8_t* dst = smem + s * Cfg::SLOT_BYTES + u * Cfg::CODE_BYTES;
          float* sc = reinterpret_cast<float*>(smem + Cfg::OFF_SCALE + s * 32 + u * 16);
          if (mine && bad) {
            // a page that is not there reads as zeros: scales of zero over whatever codes are there, or
            // zeros in the place of bf16 rows
            report_error(p.err, DEVERR_BAD_PAGE, 11, pid);
            if (q8) {
              *reinterpret_cast<float4*>(sc) = make_float4(0.f, 0.f, 0.f, 0.f);
            } else {
              for (int e = 0; e < Cfg::CODE_BYTES; e += 16) *reinterpret_cast<uint4*>(dst + e) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before later copies to the same place
          }
          __syncwarp();
          if (mine && u == 0) mbar_arrive_expect_tx(&full[s], both);
          __syncwarp();
          if (mine) {
            if (bytes && q8) {  // the scales by a plain asynchronous copy: all lanes' in one instruction
              async_copy16(sc, p.scales + block * kScalesPerBlock);
              async_copy_arrive(&full[s]);
            } else {
              mbar_arrive(&full[s]);
            }
          }
          if (mine && bytes) {
            if (q8) {
              bulk_load_hint(dst, p.codes + block * Cfg::CODE_BYTES, Cfg::CODE_BYTES, &full[s], pol);
            } else {
#pragma unroll
              for (int h = 0; h < Cfg::HALVES; ++h)
                tma_load_4d_hint(dst + h * Cfg::TILE_BYTES, u ? &tmv : &tmk, &full[s], h * 64, x.hk, 0, pid, pol);
            }
          }
          gs += min(Cfg::BATCH, count - k0 - i0);
        }
      }
    }
    if (!ok) {
      // a consumer never gave a slot back: wait (again with a limit) for the copies in flight
      if (lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, 11, (int)gs);
      for (uint32_t y = gs > RING ? gs - RING : 0; y < gs; ++y) mbar_wait(&full[y % RING], (y / RING) & 1u);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, c = lane & 3;
  const uint32_t k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_chunk_hi = lane >> 4;
  const uint32_t v_row = (lane & 7) + (lane >> 4) * 8, v_chunk_hi = (lane >> 3) & 1;
  uint2* sq = reinterpret_cast<uint2*>(smem + Cfg::OFF_Q) + lane;  // [KT][32]: the same for every warp
  bool failed = false;

  while (next_piece(p, share, x)) {
    // Q as f16 with a power of two per head, and (once per CTA) as it is for the bf16 pages
    uint32_t qf[KT][2];
    float q0, q1;  // what a score of heads 2 c and 2 c + 1 is multiplied by: their powers and the softmax scale
    {
      const bool valid = g < GROUP;
      const __nv_bfloat16* qrow = p.q + (int64_t)x.b * p.q_stride_tok + (int64_t)(x.hk * GROUP + (valid ? g : 0)) * D;
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < KT; ++j) {  // all loads before the first store, which they could not pass
        qf[j][0] = valid ? *reinterpret_cast<const uint32_t*>(qrow + 16 * j + 2 * c) : 0u;
        qf[j][1] = valid ? *reinterpret_cast<const uint32_t*>(qrow + 16 * j + 2 * c + 8) : 0u;
      }
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        if (warp == j % kNW) sq[j * 32] = make_uint2(qf[j][0], qf[j][1]);
#pragma unroll
        for (int t = 0; t < 2; ++t) top = fmaxf(top, fmaxf(fabsf(bf16_lo(qf[j][t])), fabsf(bf16_hi(qf[j][t]))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e <= top < 2^(e + 1), within the powers whose reciprocals are ordinary numbers
      const int e = min(max((int)(__float_as_uint(top) >> 23), 2), 252);
      const float down = __uint_as_float((uint32_t)(254 - e) << 23), up = __uint_as_float((uint32_t)e << 23);
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) qf[j][t] = pack_f16(bf16_lo(qf[j][t]) * down, bf16_hi(qf[j][t]) * down);
      q0 = __shfl_sync(0xffffffffu, up, 8 * c) * p.scale_log2;
      q1 = __shfl_sync(0xffffffffu, up, 8 * c + 4) * p.scale_log2;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kNW * 32));  // sq is written
    float o[KT][4];
#pragma unroll
    for (int k = 0; k < KT; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    // raises the running maxima to those of the new scores and rescales what is summed so far; r0, r1: what a
    // weight's exponent has to lose
    auto raise = [&](float t0, float t1, float& r0, float& r1) {
      const float n0 = fmaxf(m0, max_over_rows(t0)), n1 = fmaxf(m1, max_over_rows(t1));
      if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
        // (the sums in two steps: they may be 2^105, of zero blocks, so that a factor below fp32's least still counts)
        const float h0 = m0 == n0 ? 1.f : ex2_approx(0.5f * (m0 - n0)), h1 = m1 == n1 ? 1.f : ex2_approx(0.5f * (m1 - n1));
        const float a0 = h0 * h0, a1 = h1 * h1;
        m0 = n0;
        m1 = n1;
        l0 = l0 * h0 * h0;
        l1 = l1 * h1 * h1;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          o[k][0] *= a0;
          o[k][1] *= a1;
          o[k][2] *= a0;
          o[k][3] *= a1;
        }
      }
      r0 = (m0 == -INFINITY ? 0.f : m0) - kWeightLog2;  // no score above -inf: weights of zero, not NaN
      r1 = (m1 == -INFINITY ? 0.f : m1) - kWeightLog2;
    };

    const int count = x.s1 - x.s0;
    for (int k = (warp + kNW - (int)(gs % kNW)) % kNW; k < count; k += kNW) {
      const uint32_t at = gs + k;
      const int s = (int)(at % RING);
      if (!mbar_wait(&full[s], (at / RING) & 1u)) {
        if (lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, 11, 1000000 + (int)at);
        failed = true;
        break;
      }
      const int sl = x.s0 + k;
      uint8_t* slot = smem + s * Cfg::SLOT_BYTES;
      if (sl < x.r.hs) {
        // ------------------------------------------ two 8-bit pages (or the last one): 32 keys
        const float4* scp = reinterpret_cast<const float4*>(smem + Cfg::OFF_SCALE + s * 32);
        const bool two = 2 * sl + 1 < x.r.nh;
        const int left = min(x.r.n, x.r.nh * kPageTokens) - 2 * sl * kPageTokens;  // 8-bit keys from here on, >= 1
        float sc[2][4], iv[2][2];
        bool tiny = false;  // a value scale below kMinValueScale, the same for the warp
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sd[4] = {0.f, 0.f, 0.f, 0.f};
          sc[e][0] = sc[e][1] = sc[e][2] = sc[e][3] = 0.f;
          if (e == 0 || two) {
            const uint8_t* kt = slot + e * Cfg::CODE_BYTES + lane * 16;
#pragma unroll
            for (int y = 0; y < KT / 2; ++y) {
              const uint4 v = *reinterpret_cast<const uint4*>(kt + y * 512);
              uint32_t a0, a1, a2, a3;
              codes_to_f16(v.x, a0, a2);
              codes_to_f16(v.y, a1, a3);
              mma_f16_16816(sc[e], a0, a1, a2, a3, qf[2 * y][0], qf[2 * y][1]);
              codes_to_f16(v.z, a0, a2);
              codes_to_f16(v.w, a1, a3);
              mma_f16_16816(sd, a0, a1, a2, a3, qf[2 * y + 1][0], qf[2 * y + 1][1]);
            }
          }
          float4 f = two || e == 0 ? scp[e] : make_float4(0.f, 0.f, 1.f, 1.f);
          // blocks past the row's end: whatever their scales hold
          if (16 * e >= left) f.x = 0.f, f.z = 1.f;
          if (16 * e + 8 >= left) f.y = 0.f, f.w = 1.f;
          const bool t0 = f.z < kMinValueScale, t1 = f.w < kMinValueScale;
          tiny |= t0 || t1;
          const float v0 = t0 ? kMinValueScale : f.z, v1 = t1 ? kMinValueScale : f.w;
          const float g0 = lg2_approx(v0), g1 = lg2_approx(v1);
          iv[e][0] = __fdividef(1.f, v0);
          iv[e][1] = __fdividef(1.f, v1);
          sc[e][0] = fmaf(sc[e][0] + sd[0], f.x * q0, g0);
          sc[e][1] = fmaf(sc[e][1] + sd[1], f.x * q1, g0);
          sc[e][2] = fmaf(sc[e][2] + sd[2], f.y * q0, g1);
          sc[e][3] = fmaf(sc[e][3] + sd[3], f.y * q1, g1);
        }
        if (left < 32) {  // keys past the row's end have no weight
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (16 * e + g + (y & 2) * 4 >= left) sc[e][y] = -INFINITY;
        }
        float r0, r1;
        raise(fmaxf(fmaxf(sc[0][0], sc[0][2]), fmaxf(sc[1][0], sc[1][2])),
              fmaxf(fmaxf(sc[0][1], sc[0][3]), fmaxf(sc[1][1], sc[1][3])), r0, r1);
        if (tiny) {  // those blocks' weights in the sum, by themselves (2^105 at most: M is no less than s - 90)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 v = *reinterpret_cast<const float2*>(&scp[e].z);  // (keys that are not there have scores of -inf)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float own = h ? v.y : v.x;
              if (own < kMinValueScale) {
                l0 += ex2_approx(sc[e][2 * h] - kMinValueScaleLog2 - r0);  // 2^(s - M)
                l1 += ex2_approx(sc[e][2 * h + 1] - kMinValueScaleLog2 - r1);
                iv[e][h] = 0.f;
                // the product's weight, of its own scale: 0 for 0, and for what lies behind the row's end
                const float less = own > 0.f ? lg2_approx(own) - kMinValueScaleLog2 : -INFINITY;
                sc[e][2 * h] += less;
                sc[e][2 * h + 1] += less;
              }
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            sc[e][y] = ex2_approx(sc[e][y] - (y & 1 ? r1 : r0));
            if (y & 1) l1 = fmaf(sc[e][y], iv[e][y >> 1], l1);
            else l0 = fmaf(sc[e][y], iv[e][y >> 1], l0);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e == 1 && !two) break;
          const uint32_t pb0 = movmatrix_trans(pack_f16(sc[e][0], sc[e][1]));
          const uint32_t pb1 = movmatrix_trans(pack_f16(sc[e][2], sc[e][3]));
          const uint8_t* vt = slot + e * Cfg::CODE_BYTES + kPageTokens * D + lane * 16;
#pragma unroll
          for (int y = 0; y < KT / 2; ++y) {
            const uint4 v = *reinterpret_cast<const uint4*>(vt + y * 512);
            uint32_t a0, a1, a2, a3;
            codes_to_f16(v.x, a0, a1);
            codes_to_f16(v.y, a2, a3);
            mma_f16_16816(o[2 * y], a0, a1, a2, a3, pb0, pb1);
            codes_to_f16(v.z, a0, a1);
            codes_to_f16(v.w, a2, a3);
            mma_f16_16816(o[2 * y + 1], a0, a1, a2, a3, pb0, pb1);
          }
        }
      } else {
        // ------------------------------------------ one bf16 page: 16 keys
        uint8_t* vt = slot + Cfg::CODE_BYTES;
        const uint32_t kbase = smem_u32(slot), vbase = smem_u32(vt);
        float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          uint32_t a0, a1, a2, a3;
          ldmatrix_x4(a0, a1, a2, a3, kbase + (j >> 2) * Cfg::TILE_BYTES + swz128(k_row, 2 * (j & 3) + k_chunk_hi));
          const uint2 b = sq[j * 32];
          if (j & 1) mma_bf16_16816(sd, a0, a1, a2, a3, b.x, b.y);
          else mma_bf16_16816(sc, a0, a1, a2, a3, b.x, b.y);
        }
        const int left = x.r.n - (x.r.nh + sl - x.r.hs) * kPageTokens;  // >= 1
#pragma unroll
        for (int y = 0; y < 4; ++y)
          sc[y] = g + (y & 2) * 4 < left ? (sc[y] + sd[y]) * p.scale_log2 : -INFINITY;
        float r0, r1;
        raise(fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3]), r0, r1);
#pragma unroll
        for (int y = 0; y < 4; ++y) sc[y] = ex2_approx(sc[y] - (y & 1 ? r1 : r0));
        l0 += sc[0] + sc[2];
        l1 += sc[1] + sc[3];
        const uint32_t pb0 = movmatrix_trans(pack_bf16(sc[0], sc[1]));
        const uint32_t pb1 = movmatrix_trans(pack_bf16(sc[2], sc[3]));
        if (left < kPageTokens) {  // rows past the end may hold NaN: 0 * NaN would reach O
          const int per = (kPageTokens - left) * 8;
          for (int e = lane; e < per * Cfg::HALVES; e += 32) {
            const int rem = e % per;
            *reinterpret_cast<uint4*>(vt + e / per * Cfg::TILE_BYTES + (left + rem / 8) * 128 + rem % 8 * 16) =
                make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the slot's next copy
          __syncwarp();
        }
#pragma unroll
        for (int y = 0; y < KT; ++y) {
          uint32_t a0, a1, a2, a3;
          ldmatrix_x4_trans(a0, a1, a2, a3,
                            vbase + (y >> 2) * Cfg::TILE_BYTES + swz128(v_row, 2 * (y & 3) + v_chunk_hi));
          mma_bf16_16816(o[y], a0, a1, a2, a3, pb0, pb1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    gs += count;

    // ------------------------------------------------------------ the piece's partial
    // Only consumer warps write the failure flag, and only before the first barrier.
    l0 = sum_over_rows(l0);
    l1 = sum_over_rows(l1);
    if (failed && lane == 0) *fail_flag = 1;
    if (g == 0) {
      jm[warp * 8 + 2 * c] = m0;
      jm[warp * 8 + 2 * c + 1] = m1;
      jl[warp * 8 + 2 * c] = l0;
      jl[warp * 8 + 2 * c + 1] = l1;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kNW * 32));
    if (*fail_flag) return;  // the same for all consumer warps
    // every warp brings its sums to the maximum of all of them
    auto factor = [&](int h, float own) {
      float M = jm[h];
#pragma unroll
      for (int v = 1; v < kNW; ++v) M = fmaxf(M, jm[v * 8 + h]);
      return own == M ? 1.f : ex2_approx(own - M);
    };
    const float f0 = factor(2 * c, m0), f1 = factor(2 * c + 1, m1);
    // two heads at a time: thread (g, c) holds heads 2c and 2c + 1
#pragma unroll 1
    for (int hc = 0; hc < (GROUP + 1) / 2; ++hc) {
      if (c == hc) {
        float* w0 = jo + warp * 2 * Cfg::OSTRIDE;
        float* w1 = w0 + Cfg::OSTRIDE;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          w0[16 * k + g] = o[k][0] * f0;
          w1[16 * k + g] = o[k][1] * f1;
          w0[16 * k + g + 8] = o[k][2] * f0;
          w1[16 * k + g + 8] = o[k][3] * f1;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kNW * 32));
      constexpr int HC = GROUP < 2 ? GROUP : 2;
      for (int idx = threadIdx.x; idx < HC * D / 2; idx += kNW * 32) {
        const int hl = idx / (D / 2), d = idx % (D / 2) * 2, h = 2 * hc + hl;
        float M = jm[h];
#pragma unroll
        for (int v = 1; v < kNW; ++v) M = fmaxf(M, jm[v * 8 + h]);
        float L = 0.f;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < kNW; ++v) {
          const float m = jm[v * 8 + h], half = m == M ? 1.f : ex2_approx(0.5f * (m - M));
          L = fmaf(jl[v * 8 + h] * half, half, L);
          const float2 part = *reinterpret_cast<const float2*>(jo + (v * 2 + hl) * Cfg::OSTRIDE + d);
          acc.x += part.x;
          acc.y += part.y;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;  // no key: zeros; a NaN stays one
        const float lse = L == 0.f ? -INFINITY : (M + log2f(L) - kWeightLog2) * 0.6931471805599453f;
        if (p.whole) {  // the result
          const int hq = x.hk * GROUP + h;
          const float f = p.out_scale ? p.out_scale[hq] * inv : inv;
          *reinterpret_cast<uint32_t*>(p.out + (int64_t)x.b * p.out_stride_tok + (int64_t)hq * D + d) =
              pack_bf16(acc.x * f, acc.y * f);
          if (p.lse && d == 0) p.lse[(int64_t)x.b * p.Hq + hq] = lse;
        } else {
          const int64_t at = (int64_t)x.id * GROUP + h;
          *reinterpret_cast<float2*>(p.part_o + at * D + d) = make_float2(acc.x * inv, acc.y * inv);
          if (d == 0) p.part_lse[at] = lse;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kNW * 32));  // the area is rewritten
    }
  }
}

// The exact join of a (row, query head)'s pieces, times out_scale.  WARPS warps take a row's pieces by turns: one
// where there are many rows, with few pieces each, 8 where there are few.
template <int D, int WARPS>
__global__ void __launch_bounds__(256) join_pieces_kernel(const DecodeQ8Params p, int group) {
  constexpr int PER = D / 32;
  __shared__ float part[WARPS > 1 ? 8 : 1][D + 2];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = WARPS > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
  const int turn = WARPS > 1 ? warp : 0;
  if (row >= (int64_t)p.B * p.Hq) return;
  const int b = (int)(row / p.Hq), h = (int)(row % p.Hq), hk = h / group;
  const int slots = row_of(p, b).slots;
  const unsigned per = p.first_place[p.B];
  const unsigned from = p.first_place[b] + hk * (slots + kPieceCost) + kPieceCost;  // the first slot's place
  const int cta = (int)(from / per), count = slots ? (int)((from + slots - 1) / per) - cta + 1 : 0;
  const int64_t first = b * p.Hkv + hk + cta;
  const float* o = p.part_o + (first * group + h % group) * D + lane * PER;
  const float* lse = p.part_lse + first * group + h % group;
  float M = -INFINITY, L = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  constexpr int C = 8;  // pieces whose parts are requested together
  auto weight = [&M](float ls) { return ls == M ? 1.f : exp2f((ls - M) * 1.4426950408889634f); };
  for (int i0 = turn; i0 < count; i0 += C * WARPS) {
    float v[C][PER], ls[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int at = i0 + i * WARPS;
      const bool have = at < count;
      ls[i] = have ? __ldcg(lse + (int64_t)at * group) : -INFINITY;
      const float* src = o + (int64_t)(have ? at : i0) * group * D;
      if constexpr (PER == 4) {
        const float4 t = __ldcg(reinterpret_cast<const float4*>(src));
        v[i][0] = t.x, v[i][1] = t.y, v[i][2] = t.z, v[i][3] = t.w;
      } else {
        const float2 t = __ldcg(reinterpret_cast<const float2*>(src));
        v[i][0] = t.x, v[i][1] = t.y;
      }
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < C; ++i) top = fmaxf(top, ls[i]);
    const float keep = M == top ? 1.f : exp2f((M - top) * 1.4426950408889634f);
    M = top;
    L *= keep;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] *= keep;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (ls[i] == -INFINITY) continue;  // no keys
      const float w = weight(ls[i]);     // NaN where ls is
      L += w;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] = fmaf(w, v[i][e], acc[e]);
    }
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int e = 0; e < PER; ++e) part[warp][lane * PER + e] = acc[e];
    if (lane == 0) part[warp][D] = M, part[warp][D + 1] = L;
    __syncthreads();
    if (warp != 0) return;
    M = -INFINITY;
    L = 0.f;
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, part[w][D]);
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = 0.f;
    for (int w = 0; w < WARPS; ++w) {
      const float f = weight(part[w][D]);
      L += part[w][D + 1] * f;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] = fmaf(part[w][lane * PER + e], f, acc[e]);
    }
  }
  const float f = L == 0.f ? 0.f : (p.out_scale ? p.out_scale[h] : 1.f) / L;
  __nv_bfloat16* dst = p.out + (int64_t)b * p.out_stride_tok + (int64_t)h * D + lane * PER;
#pragma unroll
  for (int e = 0; e < PER; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16(acc[e] * f, acc[e + 1] * f);
  if (p.lse && lane == 0) p.lse[row] = L == 0.f ? -INFINITY : M + logf(L);
}

constexpr double kL2KeepFraction = 0.25;  // as decode_paged keeps
constexpr int kL2KeepMaxBatch = 16;

struct DevInfo {
  int sms = 0, l2 = 0;
  int occ[2][4] = {{0}};
};
DevInfo g_dev[64];
std::mutex g_mutex;

template <int D, int GROUP>
int occupancy(int dev) {
  constexpr int di = D == 128, gi = GROUP == 1 ? 0 : GROUP == 2 ? 1 : GROUP == 4 ? 2 : 3;
  std::lock_guard<std::mutex> lock(g_mutex);
  DevInfo& info = g_dev[dev];
  if (info.occ[di][gi] == 0) {
    const auto kern = decode_q8_kernel<D, GROUP>;
    int occ = 0, sms = 0, l2 = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Q8Cfg<D>::SMEM_BYTES) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, kThreads, Q8Cfg<D>::SMEM_BYTES) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&l2, cudaDevAttrL2CacheSize, dev) != cudaSuccess || occ < 1)
      return -1;
    info.sms = sms;
    info.l2 = l2;
    info.occ[di][gi] = occ;
  }
  return info.occ[di][gi];
}

template <int D, int GROUP>
int launch_q8(const CUtensorMap& tmk, const CUtensorMap& tmv, DecodeQ8Params& prm, uint8_t* ws, size_t ws_bytes,
              int dev, int keep, cudaStream_t stream) {
  const int occ = occupancy<D, GROUP>(dev);
  if (occ < 0) return LKV_ERR_CUDA;
  if (keep && prm.B <= kL2KeepMaxBatch) {
    const double page_bytes = (double)prm.Hkv * Q8Cfg<D>::CODE_BYTES;
    prm.keep_pages = (int)std::min<double>(prm.W, kL2KeepFraction * g_dev[dev].l2 / (page_bytes * prm.B));
  }
  // A CTA for every kLeastSlots slots that the tables have room for, up to two per SM.
  const int64_t units = (int64_t)prm.B * prm.Hkv, full = (int64_t)g_dev[dev].sms * occ;
  int64_t ctas = std::min<int64_t>(full, std::max<int64_t>(1, units * prm.W / kLeastSlots));
  // Short rows are not cut: without pieces there is no join launch, which costs what a CTA takes for about 40
  // slots (4 us).  The host knows the tables' width alone; `slots` is a row's as if a half of a mixed
  // table's pages were in 8 bits.
  const int64_t slots = prm.pool_pages ? (3ll * prm.W + 3) / 4 : (prm.W + 1) / 2;
  const int64_t uncut = (units + full - 1) / full * slots, cut = std::max<int64_t>(kLeastSlots, units * slots / full);
  prm.whole = slots <= 64 && uncut - cut <= 40;
  // A cut makes a piece more, which the workspace has to hold: first the rows' first places, then the pieces' lse,
  // then their o.
  const size_t piece_bytes = (size_t)GROUP * (D + 1) * sizeof(float), slack = 512;
  const size_t table = ((size_t)prm.B + 1) * sizeof(int);
  const int64_t room = ws_bytes > table + slack ? (int64_t)((ws_bytes - table - slack) / piece_bytes) : 0;
  if (room < units + ctas - 1) {
    // fewer cuts, or (with fewer CTAs than whole (row, head)s would keep busy) none
    ctas = std::min(ctas, room - units + 1);
    if (ctas < std::min(full, units)) prm.whole = 1;
  }
  if (prm.whole) ctas = std::min(full, units);
  const size_t skip = (table + 255) & ~size_t(255);
  const size_t lse_bytes = ((size_t)(units + ctas - 1) * GROUP * sizeof(float) + 255) & ~size_t(255);
  prm.first_place = reinterpret_cast<int*>(ws);
  prm.part_lse = reinterpret_cast<float*>(ws + skip);
  prm.part_o = reinterpret_cast<float*>(ws + skip + lse_bytes);
  if (launch_pdl(decode_q8_kernel<D, GROUP>, dim3((unsigned)ctas), dim3(kThreads), Q8Cfg<D>::SMEM_BYTES, stream, tmk,
                 tmv, prm) != cudaSuccess)
    return LKV_ERR_CUDA;
  if (prm.whole) return LKV_OK;
  const int64_t rows = (int64_t)prm.B * prm.Hq;
  const bool few = rows <= 4 * g_dev[dev].sms;
  const auto join = few ? join_pieces_kernel<D, 8> : join_pieces_kernel<D, 1>;
  return launch_pdl(join, dim3((unsigned)(few ? rows : (rows + 7) / 8)), dim3(256), 0, stream, prm, GROUP) ==
                 cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

}  // namespace

int decode_paged_q8(const DecodeQ8Args& a) {
  if (a.head_dim != 64 && a.head_dim != 128) return LKV_ERR_UNSUPPORTED;
  if (a.num_kv_heads <= 0 || a.num_q_heads <= 0 || a.num_q_heads % a.num_kv_heads) return LKV_ERR_INVALID_ARGUMENT;
  const int group = a.num_q_heads / a.num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8) return LKV_ERR_UNSUPPORTED;
  if (a.num_kv_heads > 256) return LKV_ERR_UNSUPPORTED;
  if (a.batch < 0 || a.max_pages_per_seq < 0 || a.max_pages_per_seq > INT_MAX / kPageTokens)
    return LKV_ERR_INVALID_ARGUMENT;
  if (a.batch == 0) return LKV_OK;
  // slots are counted in 32 bits
  if ((int64_t)a.batch * a.num_q_heads > INT_MAX / 2 ||
      (int64_t)a.batch * a.num_kv_heads * (a.max_pages_per_seq + kPieceCost) > INT_MAX) return LKV_ERR_UNSUPPORTED;
  if (!a.q || !a.codes || !a.scales || (!a.block_table && a.max_pages_per_seq) || !a.seq_k || !a.out)
    return LKV_ERR_INVALID_ARGUMENT;
  if (a.q8_pages < 0 || a.q8_pages > INT32_MAX || a.num_pages < 0 || a.num_pages > INT32_MAX)
    return LKV_ERR_INVALID_ARGUMENT;
  auto off = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; };
  if (off(a.q, 4) || (a.q_stride_tok & 1) || off(a.out, 4) || (a.out_stride_tok & 1) || off(a.codes, 16) || off(a.scales, 16))
    return LKV_ERR_INVALID_ARGUMENT;
  const int64_t row = (int64_t)a.num_q_heads * a.head_dim;
  if (a.out_stride_tok < row || a.q_stride_tok < 0) return LKV_ERR_INVALID_ARGUMENT;
  const bool pool = a.pool_k != nullptr && a.num_pages > 0;
  if (a.num_q8 && (pool != (a.pool_v != nullptr && a.num_pages > 0))) return LKV_ERR_INVALID_ARGUMENT;
  if (!a.workspace || off(a.workspace, 256) || a.workspace_bytes < kWorkspaceHeader + 256) return LKV_ERR_WORKSPACE;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LKV_ERR_CUDA;

  CUtensorMap tmk{}, tmv{};
  if (pool) {
    int st = make_pool_tensor_map(&tmk, a.pool_k, a.num_pages, a.num_kv_heads, a.head_dim);
    if (st != LKV_OK) return st;
    st = make_pool_tensor_map(&tmv, a.pool_v, a.num_pages, a.num_kv_heads, a.head_dim);
    if (st != LKV_OK) return st;
  }
  DecodeQ8Params prm{};
  prm.q = static_cast<const __nv_bfloat16*>(a.q);
  prm.q_stride_tok = a.q_stride_tok;
  prm.codes = static_cast<const uint8_t*>(a.codes);
  prm.scales = a.scales;
  prm.q8_pages = a.q8_pages;
  prm.pool_pages = pool ? a.num_pages : 0;
  prm.bt = a.block_table;
  prm.bt_stride = a.block_table_stride;
  prm.num_q8 = a.num_q8;
  prm.seq_k = a.seq_k;
  prm.out = static_cast<__nv_bfloat16*>(a.out);
  prm.out_stride_tok = a.out_stride_tok;
  prm.lse = a.lse;
  prm.out_scale = a.out_scale;
  prm.err = static_cast<int*>(a.workspace);
  prm.B = a.batch;
  prm.Hq = a.num_q_heads;
  prm.Hkv = a.num_kv_heads;
  prm.W = a.max_pages_per_seq;
  prm.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const int keep = a.flags & LKV_DECODE_L2_KEEP;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace) + kWorkspaceHeader;
  const size_t ws_bytes = a.workspace_bytes - kWorkspaceHeader;
#define LKV_Q8(DD, GG) return launch_q8<DD, GG>(tmk, tmv, prm, ws, ws_bytes, dev, keep, stream)
  if (a.head_dim == 128) {
    switch (group) {
      case 1: LKV_Q8(128, 1);
      case 2: LKV_Q8(128, 2);
      case 4: LKV_Q8(128, 4);
      default: LKV_Q8(128, 8);
    }
  } else {
    switch (group) {
      case 1: LKV_Q8(64, 1);
      case 2: LKV_Q8(64, 2);
      case 4: LKV_Q8(64, 4);
      default: LKV_Q8(64, 8);
    }
  }
#undef LKV_Q8
}

}  // namespace lkv
