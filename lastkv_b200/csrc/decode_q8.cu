// Split-KV decode over a cache whose older pages are held in 8 bits (sm_100a).
//
// Row b attends to seq_k[b] keys: its first num_q8[b] block-table columns are pages of int8 codes
// with scales (pages_q8.cuh), the rest pages of the bf16 pool.  Per KV head, with the GQA group's
// query heads folded into one tile,
//     S^T[16 keys, 8 heads] = K[16, D] Q^T        (mma m16n8k16, bf16 operands, fp32 sums)
//     s = S * key scale * softmax scale,  online softmax in fp32
//     O^T[D, 8 heads] += V^T[D, 16] (p * value scale)^T
// A code is a whole number up to 127 and exact in bf16, so the 8-bit pages' products are as exact
// as those of bf16 keys; the scales (one per 8 tokens, the rows of an accumulator) multiply fp32
// scores and weights.  p * scale is rounded to bf16, as decode_splitkv_kernel rounds p.
//
// Bound by HBM: an 8-bit page is half a bf16 page's bytes.  Work is cut into slots of equal bytes,
// one bf16 page or two 8-bit pages; an item is a (row, KV head, split) with its share of the
// slots.  The grid is persistent, CTA c taking items c, c + grid, ...: a producer warp fills a
// ring of STAGES x NW slots (a lane per copy: half a bf16 page by TMA, an 8-bit page's codes and
// its scales by two bulk copies), NW consumer warps take one slot of a stage each.  A consumer lane
// finds its operands of an 8-bit page in 16-byte pieces and turns them to bf16 in registers, 3.5
// instructions per two codes.  The splits' normalised partials are joined by merge_partials.

#include <math.h>

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
  float* part_o;           // S > 1: [S][B * Hq][D]
  float* part_lse;         // S > 1: natural log [S][B * Hq]
  int* err;
  int B, Hq, Hkv, W, S;
  float scale_log2;
  int keep_pages;  // leading columns that stay in L2
};

template <int D>
struct Q8Cfg {
  static constexpr int NW = 4;                           // consumer warps
  static constexpr int STAGES = D == 128 ? 3 : 6;        // 96 KB of slots: two CTAs per SM
  static constexpr int HALVES = D / 64;
  static constexpr int TILE_BYTES = kPageTokens * 128;   // 16 rows x 64 bf16
  static constexpr int CODE_BYTES = 2 * kPageTokens * D;  // keys and values of an 8-bit page
  static constexpr int SLOT_BYTES = 2 * CODE_BYTES;      // two 8-bit pages, or one bf16 page
  static constexpr int STAGE_BYTES = NW * SLOT_BYTES;
  static constexpr int SCALE_BYTES = STAGES * NW * 2 * 16;
  static constexpr int OSTRIDE = D + 4;
  static constexpr int OFF_SCALE = STAGES * STAGE_BYTES;
  static constexpr int OFF_MERGE = OFF_SCALE + SCALE_BYTES;
  // merge area: o [NW][4 heads][OSTRIDE], then m and l [NW][8]
  static constexpr int OFF_BAR = OFF_MERGE + NW * 4 * OSTRIDE * 4 + 2 * NW * 8 * 4;
  static constexpr int SMEM_BYTES = 1024 + OFF_BAR + 2 * STAGES * 8 + 16;
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

template <int D, int GROUP>
__global__ void __launch_bounds__((Q8Cfg<D>::NW + 1) * 32, 2)
    decode_q8_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                     const DecodeQ8Params p) {
  using Cfg = Q8Cfg<D>;
  constexpr int NW = Cfg::NW, STAGES = Cfg::STAGES, KT = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* mo = reinterpret_cast<float*>(smem + Cfg::OFF_MERGE);
  float* mm = mo + NW * 4 * Cfg::OSTRIDE;
  float* ml = mm + NW * 8;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* empty = full + STAGES;
  volatile int* fail_flag = reinterpret_cast<volatile int*>(empty + STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], NW);
    }
    *fail_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();

  struct Item {
    int b, hk, split, n, npages, nh, hs, s0, s1, n_iter;
  };
  const int n_items = p.S * p.Hkv * p.B;
  auto item_at = [&](int i) {
    Item it;
    it.split = i % p.S;
    it.hk = (i / p.S) % p.Hkv;
    it.b = i / (p.S * p.Hkv);
    it.n = max(0, p.seq_k[it.b]);
    it.npages = min((int)(((int64_t)it.n + kPageTokens - 1) / kPageTokens), p.W);
    it.n = min(it.n, it.npages * kPageTokens);
    it.nh = p.num_q8 ? min(max(p.num_q8[it.b], 0), it.npages) : it.npages;
    it.hs = (it.nh + 1) / 2;  // slots of 8-bit pages, then one per bf16 page
    const int slots = it.hs + it.npages - it.nh;
    const int per = (slots + p.S - 1) / p.S;
    it.s0 = min(slots, it.split * per);
    it.s1 = min(slots, it.s0 + per);
    it.n_iter = (it.s1 - it.s0 + NW - 1) / NW;
    return it;
  };

  if (warp == NW) {
    // ------------------------------------------------------------ producer
    // Lane 2 w + u copies half u of consumer warp w's slot: an 8-bit page (its codes and scales), or
    // the keys (u = 0) or values (u = 1) of a bf16 page.
    if (p.pool_pages && lane == 0) {
      tma_prefetch_desc(&tmk);
      tma_prefetch_desc(&tmv);
    }
    const uint64_t pol_first = policy_evict_first(), pol_last = policy_evict_last();
    const int w = lane >> 1, u = lane & 1;
    uint32_t gs = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < n_items; i += gridDim.x) {
      const Item it = item_at(i);
      const int32_t* row = p.bt + (int64_t)it.b * p.bt_stride;
      // this lane's page of step k: its block-table column (-1: none) and id, read a step ahead
      auto column = [&](int k) {
        const int sl = it.s0 + k * NW + w;
        if (lane >= 2 * NW || k >= it.n_iter || sl >= it.s1) return -1;
        if (sl >= it.hs) return it.nh + sl - it.hs;
        return 2 * sl + u < it.nh ? 2 * sl + u : -1;
      };
      int col = column(0);
      int id = col >= 0 ? __ldg(row + col) : 0;
      for (int k = 0; k < it.n_iter; ++k, ++gs) {
        const int c = col, pid = id;
        col = column(k + 1);
        if (col >= 0) id = __ldg(row + col);
        const int s = (int)(gs % STAGES);
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((gs / STAGES) & 1u) ^ 1u));
        if (!ok) break;
        const bool q8 = c >= 0 && c < it.nh;
        const bool bad = c >= 0 && (pid < 0 || (int64_t)pid >= (q8 ? p.q8_pages : p.pool_pages));
        uint8_t* dst = smem + s * Cfg::STAGE_BYTES + w * Cfg::SLOT_BYTES + u * Cfg::CODE_BYTES;
        float* sc = reinterpret_cast<float*>(smem + Cfg::OFF_SCALE + (s * NW + w) * 32 + u * 16);
        uint32_t bytes = 0;
        if (c >= 0 && !bad) bytes = Cfg::CODE_BYTES + (q8 ? 16 : 0);
        if (bad) {
          // a page that is not there reads as zeros: scales of zero over whatever codes are there,
          // or zeros in the place of bf16 rows
          report_error(p.err, DEVERR_BAD_PAGE, 11, pid);
          if (q8) {
            *reinterpret_cast<float4*>(sc) = make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            for (int e = 0; e < Cfg::CODE_BYTES; e += 16) *reinterpret_cast<uint4*>(dst + e) = make_uint4(0, 0, 0, 0);
          }
          // before later copies into the same place
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        const uint32_t total = __reduce_add_sync(0xffffffffu, bytes);
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(&full[s], total);
        __syncwarp();
        if (bytes) {
          const uint64_t pol = c < p.keep_pages ? pol_last : pol_first;
          if (q8) {
            const int64_t block = (int64_t)pid * p.Hkv + it.hk;
            bulk_load_hint(dst, p.codes + block * Cfg::CODE_BYTES, Cfg::CODE_BYTES, &full[s], pol);
            bulk_load(sc, p.scales + block * kScalesPerBlock, 16, &full[s]);
          } else {
#pragma unroll
            for (int h = 0; h < Cfg::HALVES; ++h)
              tma_load_4d_hint(dst + h * Cfg::TILE_BYTES, u ? &tmv : &tmk, &full[s], h * 64, it.hk, 0, pid, pol);
          }
        }
      }
    }
    if (!ok) {
      // a consumer never gave a slot back: wait (again with a limit) for the copies in flight
      if (lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, 11, (int)gs);
      for (uint32_t x = gs > STAGES ? gs - STAGES : 0; x < gs; ++x) mbar_wait(&full[x % STAGES], (x / STAGES) & 1u);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, c = lane & 3;
  const uint32_t k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_chunk_hi = lane >> 4;
  const uint32_t v_row = (lane & 7) + (lane >> 4) * 8, v_chunk_hi = (lane >> 3) & 1;
  uint32_t gs = 0;
  bool failed = false;

  for (int i = blockIdx.x; i < n_items; i += gridDim.x) {
    const Item it = item_at(i);
    uint32_t qf[KT][2];
    {
      const bool valid = g < GROUP;
      const __nv_bfloat16* qrow =
          p.q + (int64_t)it.b * p.q_stride_tok + (int64_t)(it.hk * GROUP + (valid ? g : 0)) * D;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        const int d0 = 16 * j + 2 * c;
        qf[j][0] = valid ? *reinterpret_cast<const uint32_t*>(qrow + d0) : 0u;
        qf[j][1] = valid ? *reinterpret_cast<const uint32_t*>(qrow + d0 + 8) : 0u;
      }
    }
    float o[KT][4];
#pragma unroll
    for (int k = 0; k < KT; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    // raises the running maxima to the new scores' and rescales what is summed so far
    auto raise = [&](float t0, float t1, float& r0, float& r1) {
      const float n0 = fmaxf(m0, max_over_rows(t0)), n1 = fmaxf(m1, max_over_rows(t1));
      if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
        const float a0 = m0 == n0 ? 1.f : ex2_approx(m0 - n0), a1 = m1 == n1 ? 1.f : ex2_approx(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          o[k][0] *= a0;
          o[k][1] *= a1;
          o[k][2] *= a0;
          o[k][3] *= a1;
        }
      }
      r0 = m0 == -INFINITY ? 0.f : m0;  // no score above -inf: weights of zero, not NaN
      r1 = m1 == -INFINITY ? 0.f : m1;
    };

    for (int k = 0; k < it.n_iter; ++k, ++gs) {
      const int s = (int)(gs % STAGES);
      if (!mbar_wait(&full[s], (gs / STAGES) & 1u)) {
        if (lane == 0) report_error(p.err, DEVERR_WAIT_TIMEOUT, 11, 1000000 + (int)gs);
        failed = true;
        break;
      }
      const int sl = it.s0 + k * NW + warp;
      uint8_t* slot = smem + s * Cfg::STAGE_BYTES + warp * Cfg::SLOT_BYTES;
      if (sl < it.s1 && sl < it.hs) {
        // ------------------------------------------ two 8-bit pages (or the last one): 32 keys
        const float4* scp = reinterpret_cast<const float4*>(smem + Cfg::OFF_SCALE + (s * NW + warp) * 32);
        const bool two = 2 * sl + 1 < it.nh;
        const int left = min(it.n, it.nh * kPageTokens) - 2 * sl * kPageTokens;  // 8-bit keys from here on, >= 1
        float sc[2][4], pv[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sd[4] = {0.f, 0.f, 0.f, 0.f};
          sc[e][0] = sc[e][1] = sc[e][2] = sc[e][3] = 0.f;
          if (e == 0 || two) {
            const uint8_t* kt = slot + e * Cfg::CODE_BYTES + lane * 16;
#pragma unroll
            for (int x = 0; x < KT / 2; ++x) {
              const uint4 v = *reinterpret_cast<const uint4*>(kt + x * 512);
              uint32_t a0, a1, a2, a3;
              codes_to_bf16(v.x, a0, a2);
              codes_to_bf16(v.y, a1, a3);
              mma_bf16_16816(sc[e], a0, a1, a2, a3, qf[2 * x][0], qf[2 * x][1]);
              codes_to_bf16(v.z, a0, a2);
              codes_to_bf16(v.w, a1, a3);
              mma_bf16_16816(sd, a0, a1, a2, a3, qf[2 * x + 1][0], qf[2 * x + 1][1]);
            }
          }
          const float4 f = two || e == 0 ? scp[e] : make_float4(0.f, 0.f, 0.f, 0.f);
          const float k0 = f.x * p.scale_log2, k1 = f.y * p.scale_log2;
          sc[e][0] = (sc[e][0] + sd[0]) * k0;
          sc[e][1] = (sc[e][1] + sd[1]) * k0;
          sc[e][2] = (sc[e][2] + sd[2]) * k1;
          sc[e][3] = (sc[e][3] + sd[3]) * k1;
          pv[e][0] = pv[e][1] = f.z;
          pv[e][2] = pv[e][3] = f.w;
        }
        if (left < 32) {  // keys past the row's end: no weight, whatever they and their scales hold
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (16 * e + g + (x & 2) * 4 >= left) {
                sc[e][x] = -INFINITY;
                pv[e][x] = 0.f;
              }
        }
        float r0, r1;
        raise(fmaxf(fmaxf(sc[0][0], sc[0][2]), fmaxf(sc[1][0], sc[1][2])),
              fmaxf(fmaxf(sc[0][1], sc[0][3]), fmaxf(sc[1][1], sc[1][3])), r0, r1);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float w = ex2_approx(sc[e][x] - (x & 1 ? r1 : r0));
            if (x & 1) l1 += w;
            else l0 += w;
            pv[e][x] *= w;
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e == 1 && !two) break;
          const uint32_t pb0 = movmatrix_trans(pack_bf16(pv[e][0], pv[e][1]));
          const uint32_t pb1 = movmatrix_trans(pack_bf16(pv[e][2], pv[e][3]));
          const uint8_t* vt = slot + e * Cfg::CODE_BYTES + kPageTokens * D + lane * 16;
#pragma unroll
          for (int x = 0; x < KT / 2; ++x) {
            const uint4 v = *reinterpret_cast<const uint4*>(vt + x * 512);
            uint32_t a0, a1, a2, a3;
            codes_to_bf16(v.x, a0, a1);
            codes_to_bf16(v.y, a2, a3);
            mma_bf16_16816(o[2 * x], a0, a1, a2, a3, pb0, pb1);
            codes_to_bf16(v.z, a0, a1);
            codes_to_bf16(v.w, a2, a3);
            mma_bf16_16816(o[2 * x + 1], a0, a1, a2, a3, pb0, pb1);
          }
        }
      } else if (sl < it.s1) {
        // ------------------------------------------ one bf16 page: 16 keys
        uint8_t* vt = slot + Cfg::CODE_BYTES;
        const uint32_t kbase = smem_u32(slot), vbase = smem_u32(vt);
        float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          uint32_t a0, a1, a2, a3;
          ldmatrix_x4(a0, a1, a2, a3, kbase + (j >> 2) * Cfg::TILE_BYTES + swz128(k_row, 2 * (j & 3) + k_chunk_hi));
          if (j & 1) mma_bf16_16816(sd, a0, a1, a2, a3, qf[j][0], qf[j][1]);
          else mma_bf16_16816(sc, a0, a1, a2, a3, qf[j][0], qf[j][1]);
        }
        const int left = it.n - (it.nh + sl - it.hs) * kPageTokens;  // >= 1
#pragma unroll
        for (int x = 0; x < 4; ++x)
          sc[x] = g + (x & 2) * 4 < left ? (sc[x] + sd[x]) * p.scale_log2 : -INFINITY;
        float r0, r1;
        raise(fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3]), r0, r1);
        const float p00 = ex2_approx(sc[0] - r0), p01 = ex2_approx(sc[1] - r1);
        const float p10 = ex2_approx(sc[2] - r0), p11 = ex2_approx(sc[3] - r1);
        l0 += p00 + p10;
        l1 += p01 + p11;
        const uint32_t pb0 = movmatrix_trans(pack_bf16(p00, p01));
        const uint32_t pb1 = movmatrix_trans(pack_bf16(p10, p11));
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
        for (int x = 0; x < KT; ++x) {
          uint32_t a0, a1, a2, a3;
          ldmatrix_x4_trans(a0, a1, a2, a3,
                            vbase + (x >> 2) * Cfg::TILE_BYTES + swz128(v_row, 2 * (x & 3) + v_chunk_hi));
          mma_bf16_16816(o[x], a0, a1, a2, a3, pb0, pb1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }

    // ------------------------------------------------------------ item merge
    // Only consumer warps write the failure flag, and only before this barrier.
    l0 = sum_over_rows(l0);
    l1 = sum_over_rows(l1);
    if (failed && lane == 0) *fail_flag = 1;
    if (g == 0) {
      mm[warp * 8 + 2 * c] = m0;
      mm[warp * 8 + 2 * c + 1] = m1;
      ml[warp * 8 + 2 * c] = l0;
      ml[warp * 8 + 2 * c + 1] = l1;
    }
    // four heads at a time: thread (g, c) holds heads 2c and 2c + 1
#pragma unroll
    for (int hc = 0; hc < (GROUP + 3) / 4; ++hc) {
      if ((c >> 1) == hc) {
        float* w0 = mo + (warp * 4 + 2 * c - 4 * hc) * Cfg::OSTRIDE;
        float* w1 = w0 + Cfg::OSTRIDE;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          w0[16 * k + g] = o[k][0];
          w1[16 * k + g] = o[k][1];
          w0[16 * k + g + 8] = o[k][2];
          w1[16 * k + g + 8] = o[k][3];
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(NW * 32));
      if (*fail_flag) return;  // the same for all consumer warps
      constexpr int HC = GROUP < 4 ? GROUP : 4;
      for (int idx = threadIdx.x; idx < HC * D; idx += NW * 32) {
        const int hl = idx / D, d = idx % D, h = 4 * hc + hl;
        float M = -INFINITY;
#pragma unroll
        for (int v = 0; v < NW; ++v) M = fmaxf(M, mm[v * 8 + h]);
        float L = 0.f, acc = 0.f;
#pragma unroll
        for (int v = 0; v < NW; ++v) {
          const float f = mm[v * 8 + h] == M ? 1.f : exp2f(mm[v * 8 + h] - M);
          L += ml[v * 8 + h] * f;
          acc += mo[(v * 4 + hl) * Cfg::OSTRIDE + d] * f;
        }
        const float val = L == 0.f ? 0.f : acc / L;  // no key: zeros; a NaN stays one
        float lse = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
        if (p.S > 1 && L != L) lse = INFINITY;  // so that the merge does not pass a NaN part over
        const int hq = it.hk * GROUP + h;
        const int64_t row = (int64_t)it.b * p.Hq + hq;
        if (p.S == 1) {
          const float f = p.out_scale ? p.out_scale[hq] : 1.f;
          p.out[(int64_t)it.b * p.out_stride_tok + (int64_t)hq * D + d] = __float2bfloat16_rn(val * f);
          if (p.lse && d == 0) p.lse[row] = lse;
        } else {
          const int64_t at = (int64_t)it.split * p.B * p.Hq + row;
          p.part_o[at * D + d] = val;
          if (d == 0) p.part_lse[at] = lse;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(NW * 32));  // the area is rewritten
    }
  }
}

constexpr int kMaxSplits = 32;
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
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kern, (Q8Cfg<D>::NW + 1) * 32, Q8Cfg<D>::SMEM_BYTES) !=
            cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&l2, cudaDevAttrL2CacheSize, dev) != cudaSuccess || occ < 1)
      return -1;
    info.sms = sms;
    info.l2 = l2;
    info.occ[di][gi] = occ;
  }
  return info.occ[di][gi];
}

// Splits for the persistent grid: the busiest CTA's slots, plus a slot's time per item for its
// merge, the ring's fill, and the merge launch where there are splits.
int choose_splits(int units, int slots, int ctas, int smax) {
  int best = 1;
  int64_t best_cost = INT64_MAX;
  smax = std::min(smax, std::max(1, slots / 4));
  for (int s = 1; s <= smax; ++s) {
    const int64_t per_cta = ((int64_t)units * s + ctas - 1) / ctas;
    const int64_t cost = per_cta * ((slots + s - 1) / s + 1) + 6 + (s > 1 ? 2 : 0);
    if (cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

template <int D, int GROUP>
int launch_q8(const CUtensorMap& tmk, const CUtensorMap& tmv, DecodeQ8Params& prm, int smax, int dev, int keep,
              cudaStream_t stream) {
  const int occ = occupancy<D, GROUP>(dev);
  if (occ < 0) return LKV_ERR_CUDA;
  const int ctas = g_dev[dev].sms * occ;
  // the host does not know how many of a row's pages are in 8 bits: as if all were
  prm.S = choose_splits(prm.B * prm.Hkv, (prm.W + 1) / 2, ctas, smax);
  if (keep && prm.B <= kL2KeepMaxBatch) {
    const double page_bytes = (double)prm.Hkv * Q8Cfg<D>::CODE_BYTES;
    prm.keep_pages = (int)std::min<double>(prm.W, kL2KeepFraction * g_dev[dev].l2 / (page_bytes * prm.B));
  }
  const int64_t items = (int64_t)prm.S * prm.Hkv * prm.B;
  if (items > INT_MAX) return LKV_ERR_UNSUPPORTED;
  return launch_pdl(decode_q8_kernel<D, GROUP>, dim3((unsigned)std::min<int64_t>(items, ctas)),
                    dim3((Q8Cfg<D>::NW + 1) * 32), Q8Cfg<D>::SMEM_BYTES, stream, tmk, tmv, prm) == cudaSuccess
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
  if ((int64_t)a.batch * a.num_kv_heads > INT_MAX / kMaxSplits) return LKV_ERR_UNSUPPORTED;
  if (!a.q || !a.codes || !a.scales || !a.block_table || !a.seq_k || !a.out) return LKV_ERR_INVALID_ARGUMENT;
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
  const int64_t rows = (int64_t)a.batch * a.num_q_heads;
  // after the error header: the splits' lse, then (256-byte aligned) their o
  const size_t per_split = (size_t)rows * (a.head_dim + 1) * sizeof(float) + 256;
  const int smax = (int)std::min<size_t>(kMaxSplits, (a.workspace_bytes - kWorkspaceHeader) / per_split);
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
  uint8_t* ws = static_cast<uint8_t*>(a.workspace) + kWorkspaceHeader;
  prm.part_lse = reinterpret_cast<float*>(ws);
  prm.part_o =
      reinterpret_cast<float*>(ws + (((size_t)rows * std::max(smax, 1) * sizeof(float) + 255) & ~size_t(255)));
  prm.err = static_cast<int*>(a.workspace);
  prm.B = a.batch;
  prm.Hq = a.num_q_heads;
  prm.Hkv = a.num_kv_heads;
  prm.W = a.max_pages_per_seq;
  prm.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  const int keep = a.flags & LKV_DECODE_L2_KEEP;
  int st = LKV_ERR_UNSUPPORTED;
#define LKV_Q8(DD, GG) st = launch_q8<DD, GG>(tmk, tmv, prm, std::max(smax, 1), dev, keep, stream); break
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
  if (st != LKV_OK || prm.S == 1) return st;
  return merge_partials(prm.part_o, prm.part_lse, prm.S, rows, a.head_dim, a.num_q_heads, rows * a.head_dim, rows,
                        a.out_scale, a.out, a.lse, stream, a.out_stride_tok);
}

}  // namespace lkv
