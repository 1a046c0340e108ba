// Chunked (varlen) prefill over the shared last-layer paged K/V pool on
// 5th-generation tensor cores (tcgen05 + TMEM), sm_100a.
//
// Reference semantics: the merged per-layer attention call of the vLLM fast
// path for prefill spans (vllm/src/lastkv/vllm/backends/rmarin_flashinfer/
// fastpath.py:643-650: FA3 varlen, block_table = bt_all[l], seqused_k,
// causal with bottom-right alignment) followed by head_scale_
// (fused_qkv.py:140-155); at the HF level the masked SDPA of
// LastKVAttention.forward (llm/src/lastkv/llm/modeling.py:124-146).  The
// non-causal form serves block attention over a shared history (Wan,
// videogen/src/lastkv/videogen/attention.py:9-32).
//
// Work unit: one CTA = two 128-row query tiles (A, B) x one KV head x one
// sequence.  Rows pack TOK = 128 / GROUP query tokens times the GROUP query
// heads that share the KV head (row r -> token r / GROUP, head r % GROUP);
// tile B holds the TOK tokens after tile A.  Every K/V block brought on chip
// serves 256 rows (the whole GQA group of 2 TOK tokens).
//
// Warp roles (384 threads; warp w runs on SM sub-partition w % 4):
//   warps 0-3  softmax + epilogue of tile A, one thread per row (TMEM lane)
//   warps 4-7  softmax + epilogue of tile B
//   warps 8,10 TMA producers of the K blocks (128 keys = 8 pages): pages 0-3
//              and 4-7 of every block, each arriving with its half of the bytes
//   warp 9     TMA producer: the Q tiles once, then the V blocks
//              (so the first S waits for 8 copies per thread, not Q + 16)
//   warp 11    TMEM allocator and MMA issuer: the whole warp runs the issue
//              loop (warp-uniform descriptors, no per-MMA rebuild) and one
//              elected lane issues every tcgen05.mma / commit
// TMEM columns: S_A [0,128), S_B [128,256), O_A [256,256+D), O_B [256+D, 256+2D).
// Per key block j the MMA thread issues, in order,
//   PV_A(j-1), S_A(j), PV_B(j-1), S_B(j)
// (S = Q K^T: A = Q, B = K, both K-major in smem; PV: A = P read from TMEM,
// B = V MN-major in smem), so while one tile's softmax runs the tensor core
// works on the other tile.  P (bf16, two per column) overwrites the first 64
// columns of its own tile's S; the next S of that tile is issued after the PV
// that reads P, and tcgen05.mma from one thread executes in issue order.
// K and V stream through separate rings (2 and 3 stages).  A bf16 tile whose
// rows are all tokens of the span is written back through shared memory (its Q
// buffer) and one TMA store per warp and 64-column half; ragged tiles and fp32
// split partials store row by row (a warp store then touches 32 rows, which cost ~2,600 cycles per tile, on
// the critical path of the CTA's last tile).  The running max is
// only raised (and O rescaled in TMEM) when a row's max grows by more than
// 2^8; otherwise exp2 is taken against the stale max, which stays exact
// because the final normalisation uses the same reference.  The softmax takes
// a quarter of its exponentials on the FMA pipe (ex2_poly2) and the rest on the
// SFU, and stores P in 32-key chunks as they are ready.
//
// Older pages in 8 bits (Q8): a row's first num_q8 pages come from a staged copy of their int8
// codes (dequantise_pages_kernel: whole numbers up to 127, exact in bf16 and f16), and the scales, one for
// every 8 keys, are applied in fp32 in the softmax.  A key scale k multiplies a group's scores: it goes into
// the maximum once per group and into the FFMA in front of the exponential.  A value scale v multiplies the
// weights that PV takes, p v = 2^(s + log2 v - m): it goes into that FFMA's addend (and into the maximum, so
// that f16 holds them), and a group's sum of them times 1 / v is its part of the row's sum.  No instruction per
// key is added.  Pages in bf16 have scales of one; in a block of both kinds they count in the maximum with the
// scale of its 8-bit values, if that is smaller: their weights are bf16, which holds what is above f16's range.
// A page is one step of PV, 16 keys, so its type is chosen page by page: staged pages have values and weights in
// f16, times 2^7, whose rounding is lost in the output's (bf16 weights are not 1 where the largest is, as they are
// without scales, and took the error from 1.0 to 1.4, in short rows 1.7, times the output's rounding); bf16
// pages bf16 weights, and where they are most of the row a second bf16 term with what the first leaves out,
// in S's other columns.  That term in every row cost 11 % of a call with a quarter of its keys in bf16.
// Two spans of 1024 tokens, 32 heads of 128 over 8, against 8192 keys and half of that: 219 us with the
// staging, 209 without (prefill_paged: 167).  The softmax of a block bounds it, as there, with the scales in its
// chain.
//
// Key splits (non-causal calls and those over 8-bit pages, S > 1): blockIdx.z = sequence * S + split and
// a CTA covers its split's share of the key blocks, writing the normalised
// fp32 partial and natural-log LSE of its rows; merge_partials_kernel then
// combines the splits exactly.  With one CTA per SM, this fills the last wave
// of a grid of few, long CTAs (Wan's block attention).

#include <math.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "pages_q8.cuh"
#include "tcgen05.cuh"

namespace lkv {

namespace {

constexpr int kBM = 128;  // rows per tile
constexpr int kTiles = 2;  // query tiles per CTA
constexpr int kBN = 128;  // keys per block
constexpr int kPageTok = 16;
constexpr int kPagesPerBlock = kBN / kPageTok;
constexpr int kWarpK = 8, kWarpV = 9, kWarpK2 = 10, kWarpMma = 11;
constexpr int kThreads = 12 * 32;
constexpr int kStagesK = 2, kStagesV = 3;
constexpr float kRescaleLog2 = 8.0f;
constexpr float kLeastPageScale = 0x1p-60f;  // Q8: bf16 pages' weights are 2^75 at most
constexpr float kWeightLog2 = 7.0f;  // Q8: weights are times 2^7, so that f16 has 2^15 for the largest
// Q8: registers of a softmax thread, and of the others, of the 168 that each was launched with (8 warps gain
// what 4 lose).  Two spans of 1024 tokens over 8192 keys, without the staging: 223 us, with 168 each 239; the scales of
// a block then fit into registers before its scores are waited for: 212, now 209 (4 bytes spilled with heads of 128).
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
constexpr int kMaxKvSplits = 8;

struct PrefillParams {
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* seq_k;
  const int32_t* cu_q;
  __nv_bfloat16* out;
  int64_t out_stride_tok;
  float* lse;
  const float* out_scale;
  int* err;
  int B, Hq, Hkv, W;
  int64_t num_pages;
  int causal;
  float scale_log2;
  int S;                 // key splits: blockIdx.z = sequence * S + split
  float* part_o;         // S > 1: fp32 partials [S][rows][D], rows = token * Hq + head
  float* part_lse;       // S > 1: natural-log LSE [S][rows]
  int64_t part_rows;     // rows per split
  int tma_out;           // S == 1 and the output map is valid: full tiles leave by TMA stores
  // Q8: staged pages b * stage_width + column, their scales by the block table's page ids
  const int32_t* num_q8;  // or null: every page
  const float* q8_scales;
  int64_t q8_pages;
  int stage_width;
  int has_pool;
};

template <int D>
struct PrefillCfg {
  static constexpr int HALVES = D / 64;
  static constexpr int Q_HALF = kBM * 128;   // [128 rows][64 bf16]
  static constexpr int KV_HALF = kBN * 128;  // [128 keys][64 bf16]
  static constexpr int Q_BYTES = HALVES * Q_HALF;  // one tile
  static constexpr int KV_BYTES = HALVES * KV_HALF;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + kTiles * Q_BYTES;
  static constexpr int OFF_V = OFF_K + kStagesK * KV_BYTES;
  static constexpr int OFF_BAR = OFF_V + kStagesV * KV_BYTES;
  static constexpr int BAR_BYTES = 512;
  // At least 120 KB so a second CTA never shares the SM (each CTA holds all 512 TMEM columns).
  static constexpr int SMEM_BYTES =
      (1024 + OFF_BAR + BAR_BYTES) > 120 * 1024 ? (1024 + OFF_BAR + BAR_BYTES) : 120 * 1024;
  // Q8: after the barriers, per softmax warp the scales of a block's 16 groups of 8 keys: key scale x
  // softmax scale, log2 of the value scale, 1 / value scale
  static constexpr int OFF_SCALE = OFF_BAR + 256;
  static constexpr int SCALE_BYTES = 8 * 3 * 16 * 4;
  static constexpr int SMEM_Q8 = 1024 + OFF_SCALE + SCALE_BYTES > SMEM_BYTES ? 1024 + OFF_SCALE + SCALE_BYTES : SMEM_BYTES;
  static_assert(SMEM_Q8 <= 227 * 1024, "shared memory");
  static constexpr uint32_t IDESC_S = umma_idesc_bf16(kBM, kBN, 0, 0);
  static constexpr uint32_t IDESC_PV = umma_idesc_bf16(kBM, D, 0, 1);
  static constexpr uint32_t IDESC_PV_F16 = umma_idesc_f16(kBM, D, 0, 1);
  static constexpr uint32_t COL_S = 0;        // + tile * kBN
  static constexpr uint32_t COL_O = 2 * kBN;  // + tile * D
};

struct Bars {
  uint64_t q_full;
  uint64_t k_full[kStagesK], k_empty[kStagesK];
  uint64_t v_full[kStagesV], v_empty[kStagesV];
  uint64_t s_full[kTiles];   // MMA -> softmax: S_t(j) complete
  uint64_t p_full[kTiles];   // softmax -> MMA: P_t(j) stored in TMEM (4 warp arrivals)
  uint64_t pv_done[kTiles];  // MMA -> softmax: PV_t(j) complete
  uint32_t tmem_addr;
  int fail;
};

static_assert(sizeof(Bars) <= 256, "the scales begin behind the barriers");

struct StageMaps {
  CUtensorMap k, v;  // Q8: the staged pages
};
struct NoStageMaps {};

// Q8: a sum against a maximum larger by -`by`.  In two steps: it may be 2^105, so that one below fp32's least still counts.
__device__ __forceinline__ float lowered(float l, float by) {
  const float half = ex2_approx(0.5f * by);
  return l * half * half;
}

// Q8: the weights of a block's groups of keys with value scales below kMinValueScale (`tiny`: their lanes) in a row's
// sum, by themselves and before the block's others, against a maximum raised to what those groups have in it (so
// 2^105 at most): the row's m, l and what O loses by that.  The scores are in TMEM still.  A call, and where no scores
// are held in registers: the same code between them and their exponentials cost every call 2-9 %, in line here 5 %
// with heads of 64 (this 2.5).
__device__ __noinline__ float3 sum_zero_groups(uint32_t tiny, uint32_t scores, const float* group_scale, int last,
                                               float m, float l) {
  float alpha0 = 1.f;
  auto each = [&](auto take) {
#pragma unroll 1
    for (uint32_t left = tiny; left; left &= left - 1) {
      const int at = __ffs(left) - 1, g = (at >> 2) * 2 + (at & 1);
      uint32_t raw[8];
      tmem_ld8(scores + 8 * g, raw);
      tmem_wait_ld();
      const float scale = group_scale[g];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * g + e <= last) take(__uint_as_float(raw[e]) * scale);
    }
  };
  float top = -INFINITY;
  each([&](float t) { top = fmaxf(top, t); });
  top += kMinValueScaleLog2;
  if (top > m + kRescaleLog2) {
    alpha0 = (m == -INFINITY) ? 0.f : ex2_approx(m - top);
    l = lowered(l, m - top);
    m = top;
  }
  const float ref = kWeightLog2 - (m == -INFINITY ? 0.f : m);
  each([&](float t) { l += ex2_approx(t + ref); });
  return make_float3(m, l, alpha0);
}

template <int D, int GROUP, bool Q8>
__global__ void __launch_bounds__(kThreads, 1)
    prefill_tcgen05_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                           const __grid_constant__ CUtensorMap tmv, const __grid_constant__ CUtensorMap tmo,
                           const PrefillParams p,
                           const __grid_constant__ std::conditional_t<Q8, StageMaps, NoStageMaps> stage) {
  using Cfg = PrefillCfg<D>;
  constexpr int TOK = kBM / GROUP;  // tokens per tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + Cfg::OFF_BAR);

  const int cta_tile = blockIdx.x, hk = blockIdx.y, b = blockIdx.z / p.S, split = blockIdx.z % p.S;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q0 = p.cu_q[b];
  const int Lq = p.cu_q[b + 1] - q0;
  const int t0 = cta_tile * kTiles * TOK;
  if (t0 >= Lq) return;
  // A trailing tile with no valid token (the last CTA of a span whose length is
  // not a multiple of the CTA's tokens) is skipped: no Q load, MMAs or softmax.
  const int ntiles = (t0 + TOK < Lq) ? kTiles : 1;
  const int n = p.seq_k[b];
  const int t_end = min(t0 + kTiles * TOK, Lq);
  int lim_max = p.causal ? n - Lq + t_end - 1 : n - 1;
  lim_max = min(lim_max, n - 1);
  // Key blocks [j0, j0 + nb) of this CTA: all visible blocks, or this split's share
  // of them (non-causal calls with S > 1).
  const int nb_all = lim_max >= 0 ? lim_max / kBN + 1 : 0;
  const int per_split = (nb_all + p.S - 1) / p.S;
  const int j0 = min(nb_all, split * per_split);
  const int nb = min(nb_all, j0 + per_split) - j0;
  if (nb == 0) {
    // no visible keys: zero output rows (and -inf LSE), as an empty softmax
    for (int r = threadIdx.x; r < kTiles * TOK * GROUP; r += kThreads) {
      const int tok = t0 + r / GROUP;
      if (tok >= Lq) continue;
      const int hq = hk * GROUP + r % GROUP;
      const int64_t row = (int64_t)(q0 + tok) * p.Hq + hq;
      if (p.S > 1) {
        float* o = p.part_o + ((int64_t)split * p.part_rows + row) * D;
        for (int d = 0; d < D; ++d) o[d] = 0.f;
        p.part_lse[(int64_t)split * p.part_rows + row] = -INFINITY;
        continue;
      }
      __nv_bfloat16* o = p.out + (int64_t)(q0 + tok) * p.out_stride_tok + (int64_t)hq * D;
      for (int d = 0; d < D; ++d) o[d] = __float2bfloat16_rn(0.f);
      if (p.lse) p.lse[row] = -INFINITY;
    }
    return;
  }
  const int npages = min((n + kPageTok - 1) / kPageTok, p.W);
  const int nh = Q8 ? (p.num_q8 ? min(max(p.num_q8[b], 0), npages) : npages) : 0;  // pages in 8 bits
  const bool two_terms = Q8 && npages - nh > nh;  // of the weights of bf16 pages

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int s = 0; s < kStagesK; ++s) {
      mbar_init(&bars->k_full[s], 2);
      mbar_init(&bars->k_empty[s], 1);
    }
    for (int s = 0; s < kStagesV; ++s) {
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->p_full[t], 4);
      mbar_init(&bars->pv_done[t], 1);
    }
    bars->fail = 0;
    fence_barrier_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(&bars->tmem_addr, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_addr;

  uint8_t* sQ = smem + Cfg::OFF_Q;
  uint8_t* sK = smem + Cfg::OFF_K;
  uint8_t* sV = smem + Cfg::OFF_V;
  const int32_t* btrow = p.bt + (int64_t)b * p.bt_stride;

  auto issue = [&] {
    // ------------------------------------------------------------ MMA issuer
    const bool leader = elect_one();
    // Descriptors of each operand's first 16-element K slice; the slices and
    // ring stages are constant offsets (16-byte units) from them.
    const uint64_t qd = umma_sdesc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t kd = umma_sdesc_sw128(smem_u32(sK), 16, 1024);
    const uint64_t vd = umma_sdesc_sw128(smem_u32(sV), Cfg::KV_HALF, 1024);
    auto issue_s = [&](int t, int j) {
      const uint64_t kb = kd + (uint64_t)(((j % kStagesK) * Cfg::KV_BYTES) >> 4);
      const uint64_t qb = qd + (uint64_t)((t * Cfg::Q_BYTES) >> 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint32_t oq = ((ks >> 2) * Cfg::Q_HALF + (ks & 3) * 32) >> 4;
        const uint32_t okv = ((ks >> 2) * Cfg::KV_HALF + (ks & 3) * 32) >> 4;
        if (leader) umma_bf16_ss(tmem + Cfg::COL_S + t * kBN, qb + oq, kb + okv, Cfg::IDESC_S, ks > 0 ? 1u : 0u);
      }
      if (leader) umma_commit(&bars->s_full[t]);
    };
    auto issue_pv = [&](int t, int j) {
      const uint64_t vb = vd + (uint64_t)(((j % kStagesV) * Cfg::KV_BYTES) >> 4);
      if constexpr (Q8) {  // a page, 16 keys, is one step: f16 weights and codes, or two bf16 terms of the weights
        const int staged = nh - (j0 + j) * kPagesPerBlock;
        const uint32_t d = tmem + Cfg::COL_O + t * D, w = tmem + Cfg::COL_S + t * kBN;
#pragma unroll
        for (int ks = 0; ks < kBN / 16; ++ks) {
          const uint64_t v = vb + (uint64_t)((ks * (kPageTok * 128)) >> 4);
          const bool f16 = ks < staged;
          if (leader) umma_bf16_ts(d, w + ks * 8, v, f16 ? Cfg::IDESC_PV_F16 : Cfg::IDESC_PV, (j > 0 || ks > 0) ? 1u : 0u);
          if (leader && !f16 && two_terms) umma_bf16_ts(d, w + kBN / 2 + ks * 8, v, Cfg::IDESC_PV, 1u);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < kBN / 16; ++ks)
          if (leader)
            umma_bf16_ts(tmem + Cfg::COL_O + t * D, tmem + Cfg::COL_S + t * kBN + ks * 8,
                         vb + (uint64_t)((ks * (kPageTok * 128)) >> 4), Cfg::IDESC_PV, (j > 0 || ks > 0) ? 1u : 0u);
      }
      if (leader) umma_commit(&bars->pv_done[t]);
    };
    // Wait results are made warp-uniform so the whole warp leaves together.
    bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->q_full, 0));
    for (int j = 0; ok && j <= nb; ++j) {
      // PV_A(j-1), S_A(j), PV_B(j-1), S_B(j)
      if (j < nb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->k_full[j % kStagesK], (j / kStagesK) & 1));
        tc_fence_after();
        if (!ok) break;
      }
      if (j > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_full[(j - 1) % kStagesV], ((j - 1) / kStagesV) & 1));
        if (!ok) break;
      }
      for (int t = 0; t < ntiles; ++t) {
        if (j > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&bars->p_full[t], (j - 1) & 1));
          tc_fence_after();
          if (!ok) break;
          issue_pv(t, j - 1);
        }
        if (j < nb) issue_s(t, j);
      }
      if (!ok) break;
      if (leader) {
        if (j < nb) umma_commit(&bars->k_empty[j % kStagesK]);
        if (j > 0) umma_commit(&bars->v_empty[(j - 1) % kStagesV]);
      }
    }
    if (!ok && leader) {
      report_error(p.err, DEVERR_WAIT_TIMEOUT, 4, 100);
      bars->fail = 1;
    }
  };
  // (the bf16 kernel's roles lie side by side: nested as in the other one, they cost it 0.5 %)
  if (Q8 ? warp >= kTiles * 4 : warp == kWarpK || warp == kWarpK2 || warp == kWarpV) {
    if constexpr (Q8) regs_dec<kOtherRegs>();
    if (!Q8 || warp != kWarpMma) {
      // ------------------------------------------------------------ producers
      if (lane == 0) {
        const bool is_k = warp != kWarpV;
        const int stages = is_k ? kStagesK : kStagesV;
        const CUtensorMap* map = is_k ? &tmk : &tmv;
        const int pg0 = warp == kWarpK2 ? kPagesPerBlock / 2 : 0;
        const int npg = is_k ? kPagesPerBlock / 2 : kPagesPerBlock;
        tma_prefetch_desc(map);
        if (!is_k) {
          tma_prefetch_desc(&tmq);
          mbar_arrive_expect_tx(&bars->q_full, ntiles * Cfg::Q_BYTES);
          for (int t = 0; t < ntiles; ++t)
#pragma unroll
            for (int h = 0; h < Cfg::HALVES; ++h)
              tma_load_3d(sQ + t * Cfg::Q_BYTES + h * Cfg::Q_HALF, &tmq, &bars->q_full, h * 64, hk * GROUP,
                          q0 + t0 + t * TOK);
        }
        uint64_t* full = is_k ? bars->k_full : bars->v_full;
        uint64_t* empty = is_k ? bars->k_empty : bars->v_empty;
        uint8_t* ring = is_k ? sK : sV;
        for (int j = 0; j < nb; ++j) {
          const int s = j % stages;
          if (!mbar_wait(&empty[s], ((j / stages) & 1) ^ 1)) {
            report_error(p.err, DEVERR_WAIT_TIMEOUT, 4, j);
            bars->fail = 1;
            break;
          }
          mbar_arrive_expect_tx(&full[s], npg * (Cfg::KV_BYTES / kPagesPerBlock));
          uint8_t* dst = ring + s * Cfg::KV_BYTES;
          for (int pg = pg0; pg < pg0 + npg; ++pg) {
            const int pi = (j0 + j) * kPagesPerBlock + pg;
            int pid = (int)p.num_pages;  // past the pool: TMA fills zeros
            const CUtensorMap* from = map;
            if (Q8 && pi < nh) {
              if constexpr (Q8) from = is_k ? &stage.k : &stage.v;
              // a page without a place in the stage reads as zeros
              pid = pi < p.stage_width ? b * p.stage_width + pi : p.B * p.stage_width;
              if (is_k && pi >= p.stage_width) report_error(p.err, DEVERR_BAD_PAGE, 4, pi);
            } else if (pi < npages) {
              pid = btrow[pi];
              // (only the K producers check it: with the checks in front of every V copy, too, spans over bf16 pages
              // took 4-7 % longer; ids outside the map read as zeros by themselves)
              if (is_k && (pid < 0 || (int64_t)pid >= p.num_pages || (Q8 && !p.has_pool)))
                report_error(p.err, DEVERR_BAD_PAGE, 4, pid);
              if (Q8 && !p.has_pool) pid = (int)p.num_pages;
            }
#pragma unroll
            for (int h = 0; h < Cfg::HALVES; ++h)
              tma_load_4d(dst + h * Cfg::KV_HALF + pg * (kPageTok * 128), from, &full[s], h * 64, hk, 0, pid);
          }
        }
      }
    } else {
      issue();
    }
  } else if (!Q8 && warp == kWarpMma) {
    issue();
  } else if ((warp >> 2) < ntiles) {
    if constexpr (Q8) regs_inc<kSoftmaxRegs>();
    // ------------------------------------------------------------ softmax (rows)
    const int t = warp >> 2;                       // tile
    const int r = (warp & 3) * 32 + lane;          // TMEM lane = row within the tile
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t col_s = Cfg::COL_S + t * kBN, col_o = Cfg::COL_O + t * D;
    const int tok = t0 + t * TOK + r / GROUP;
    int lim = p.causal ? n - Lq + tok : n - 1;
    lim = min(lim, n - 1);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const float sl2 = p.scale_log2;
    float* group_scale = reinterpret_cast<float*>(smem + Cfg::OFF_SCALE) + warp * 48;  // Q8
    auto load4 = [](const float* p) {
      const uint4 v = ld_shared16(p);
      return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    };
    // Q8: lane 4 i + c has scale c (keys 0-7, 8-15, values 0-7, 8-15) of page i of a block.  It is read a block
    // ahead, and the page's id two, so that neither is waited for.
    auto page_of = [&](int j) {
      const int pi = (j0 + j) * kPagesPerBlock + (lane >> 2);
      return j < nb && pi < nh && pi < p.stage_width ? btrow[pi] : -1;
    };
    auto scale_of = [&](int pid) {
      return pid >= 0 && (int64_t)pid < p.q8_pages
                 ? __ldg(p.q8_scales + ((int64_t)pid * p.Hkv + hk) * 4 + (lane & 3)) : 1.f;
    };
    float next_scale = Q8 ? scale_of(page_of(0)) : 1.f;
    int next_page = Q8 ? page_of(1) : 0;
    // Wait results are made warp-uniform: tcgen05.ld/st below are warp-collective.
    for (int j = 0; j < nb; ++j) {
      float4 kf[4], lv[4];  // Q8
      uint32_t tiny = 0;    // Q8: the lanes whose value scale is below kMinValueScale
      if constexpr (Q8) {
        float f = next_scale;
        next_scale = scale_of(next_page);
        next_page = page_of(j + 2);
        if (!(fabsf(f) < INFINITY)) f = 1.f;  // the staged keys are NaN there
        const int at = (lane >> 2) * 2 + (lane & 1);
        const int here = nh - (j0 + j) * kPagesPerBlock;  // pages of this block in 8 bits
        if (here > 0 && here < kPagesPerBlock) {
          // both kinds: its bf16 pages count in the maximum with the scale of its 8-bit values, if that is below 1
          float top = (lane & 2) && (lane >> 2) < here ? f : 0.f;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          if ((lane & 2) && (lane >> 2) >= here && top >= kMinValueScale) f = fminf(fmaxf(top, kLeastPageScale), 1.f);
        }
        const bool small = (lane & 2) && f < kMinValueScale;
        tiny = __ballot_sync(0xffffffffu, small);
        if (lane & 2) {
          if (small) f = kMinValueScale;
          group_scale[16 + at] = lg2_approx(f);
          group_scale[32 + at] = small ? 0.f : (lane >> 2) < here ? __fdividef(1.f, f) : 1.f;
        } else {
          group_scale[at] = fmaxf(f, 1e-37f) * sl2;  // codes of zero: not -inf * 0 where they are masked
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // those of the 16 groups, before the scores are waited for
          kf[c] = load4(group_scale + 4 * c);
          lv[c] = load4(group_scale + 16 + 4 * c);
        }
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[t], j & 1));
      tc_fence_after();
      if (!ok) break;
      const int key0 = (j0 + j) * kBN;
      float alpha0 = 1.f;  // what O has lost before its block's maximum
      if constexpr (Q8) {
        if (__builtin_expect(tiny != 0, 0)) {
          const float3 r = sum_zero_groups(tiny, lane_base + col_s, group_scale, lim - key0, m, l);
          m = r.x;
          l = r.y;
          alpha0 = r.z;
        }
      }
      // raw scores; the softmax scale is folded into one FFMA per element below
      float x[kBN];
      {
        uint32_t raw[kBN / 32][32];
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c) tmem_ld32(lane_base + col_s + c * 32, raw[c]);
        tmem_wait_ld();  // one wait for all four loads
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) x[c * 32 + e] = __uint_as_float(raw[c][e]);
      }
      if (key0 + kBN - 1 > lim) {
#pragma unroll
        for (int e = 0; e < kBN; ++e)
          if (key0 + e > lim) x[e] = -INFINITY;
      }
      float mx;
      if constexpr (Q8) {
        float gm[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          auto top8 = [&x](int e) {
            return fmaxf(fmax3f(fmax3f(x[e], x[e + 1], x[e + 2]), x[e + 3], x[e + 4]), fmax3f(x[e + 5], x[e + 6], x[e + 7]));
          };
          gm[c] = fmaxf(fmax3f(fmaf(top8(32 * c), kf[c].x, lv[c].x), fmaf(top8(32 * c + 8), kf[c].y, lv[c].y),
                               fmaf(top8(32 * c + 16), kf[c].z, lv[c].z)),
                        fmaf(top8(32 * c + 24), kf[c].w, lv[c].w));
        }
        mx = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
      } else {
        // 8 independent partial maxima (short dependency chains, three-input max), then a tree
        float mp[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) mp[u] = fmaxf(x[u], x[kBN - 8 + u]);
#pragma unroll
        for (int e = 8; e + 16 <= kBN - 8; e += 16)
#pragma unroll
          for (int u = 0; u < 8; ++u) mp[u] = fmax3f(mp[u], x[e + u], x[e + 8 + u]);
        mx = fmaxf(fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])), fmaxf(fmaxf(mp[4], mp[5]), fmaxf(mp[6], mp[7])));
        mx *= sl2;  // scale > 0, so max commutes with it
      }
      float alpha = 1.f;
      if (mx > m + kRescaleLog2) {
        alpha = (m == -INFINITY) ? 0.f : ex2_approx(m - mx);
        if constexpr (Q8) l = lowered(l, m - mx);
        m = mx;
      }
      const float neg_mref = (m == -INFINITY) ? 0.f : Q8 ? kWeightLog2 - m : -m;
      const float2 sl2v = make_float2(sl2, sl2), negm = make_float2(neg_mref, neg_mref);
      float2 sp[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      // P(j) (bf16 pairs) over the first 64 columns of this tile's S, which is fully
      // read: 16 columns per 32 keys, stored as each chunk is ready.  f32x2 FFMA /
      // FADD halve the issue slots of the scale-and-subtract and the sums; pairs 0
      // and 1 of every 8 take their exponentials on the FMA pipe, the rest on the SFU.
      if constexpr (Q8) {
        const int staged = nh - (j0 + j) * kPagesPerBlock;  // pages of this block in 8 bits
        // the weights as PV takes them: f16, or (MIXED: pages from `staged` on) bf16, with TWO what that leaves out
        auto weights = [&](auto mixed, auto two) {
          constexpr bool MIXED = decltype(mixed)::value, TWO = decltype(two)::value;
#pragma unroll
          for (int c = 0; c < kBN / 32; ++c) {
            uint32_t pc[16], rest[TWO ? 16 : 1];
            const float4 iv = load4(group_scale + 32 + 4 * c);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const bool f16 = !MIXED || 2 * c + (g >> 1) < staged;
              const float scale = (&kf[c].x)[g], add = (f16 ? (&lv[c].x)[g] : 0.f) + neg_mref;
              const float2 scalev = make_float2(scale, scale), addv = make_float2(add, add);
              float2 gs = make_float2(0.f, 0.f), pv[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int e = c * 32 + g * 8 + 2 * q;
                const float2 a = __ffma2_rn(make_float2(x[e], x[e + 1]), scalev, addv);
                pv[q] = q == (g & 1) ? ex2_poly2(a) : make_float2(ex2_approx(a.x), ex2_approx(a.y));
                gs = __fadd2_rn(gs, pv[q]);
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) pc[g * 4 + q] = f16 ? pack_f16(pv[q].x, pv[q].y) : pack_bf16(pv[q].x, pv[q].y);
              if constexpr (TWO) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const uint32_t hi = pc[g * 4 + q];
                  rest[g * 4 + q] = pack_bf16(pv[q].x - bf16_lo(hi), pv[q].y - bf16_hi(hi));
                }
              }
              const float inv = (&iv.x)[g];
              sp[g] = __ffma2_rn(gs, make_float2(inv, inv), sp[g]);
            }
            tmem_st16(lane_base + col_s + c * 16, pc);
            if constexpr (TWO) tmem_st16(lane_base + col_s + kBN / 2 + c * 16, rest);
          }
        };
        if (staged >= kPagesPerBlock) weights(std::false_type{}, std::false_type{});
        else if (two_terms) weights(std::true_type{}, std::true_type{});
        else weights(std::true_type{}, std::false_type{});
      } else {
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c) {
          uint32_t pc[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const int e = c * 32 + 2 * q;
            const float2 a = __ffma2_rn(make_float2(x[e], x[e + 1]), sl2v, negm);
            const float2 pv = (q & 7) < 2 ? ex2_poly2(a) : make_float2(ex2_approx(a.x), ex2_approx(a.y));
            sp[q & 3] = __fadd2_rn(sp[q & 3], pv);
            pc[q] = pack_bf16(pv.x, pv.y);
          }
          tmem_st16(lane_base + col_s + c * 16, pc);
        }
      }
      const float sum = ((sp[0].x + sp[0].y) + (sp[1].x + sp[1].y)) + ((sp[2].x + sp[2].y) + (sp[3].x + sp[3].y));
      l = Q8 ? l + sum : l * alpha + sum;
      if constexpr (Q8) alpha *= alpha0;
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        // O holds blocks < j once PV(j-1) is complete; rescale it in TMEM
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->pv_done[t], (j - 1) & 1));
        tc_fence_after();
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t raw[32];
          tmem_ld32(lane_base + col_o + c * 32, raw);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) raw[e] = __float_as_uint(__uint_as_float(raw[e]) * alpha);
          tmem_st32(lane_base + col_o + c * 32, raw);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->p_full[t]);
    }
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bars->pv_done[t], (nb - 1) & 1));
    tc_fence_after();
    if (!ok) {
      report_error(p.err, DEVERR_WAIT_TIMEOUT, 4, 200);
      bars->fail = 1;
    }
    // A bf16 tile whose rows are all tokens of this span leaves through shared
    // memory: each thread writes its row into the tile's Q buffer (free now: the
    // tile's last S MMA completed before its last PV) in the 128-byte-swizzled
    // layout of the Q copy, and each warp stores its 32 rows of a 64-column half
    // with one TMA copy as soon as it has written them - whole lines instead of
    // one 16-byte piece of 32 rows per warp store, and no wait for the other
    // warps.  Ragged tiles (and the fp32 split partials) store row by row.
    const bool staged = p.S == 1 && p.tma_out && t0 + (t + 1) * TOK <= Lq;
    uint8_t* swarp = sQ + t * Cfg::Q_BYTES + (warp & 3) * 32 * 128;  // this warp's 32 rows of half 0
    if (ok) {
      const int hq = hk * GROUP + r % GROUP;
      const bool valid = tok < Lq;
      // no key that this row sees: zeros (the sum is not 0 beside rows that see some: ex2_poly2's 2^-125 for each
      // masked key); a sum that is not a number stays one, in the LSE too, by which the splits are merged
      const bool none = l == 0.f || (m == -INFINITY && l == l);
      const float inv = none ? 0.f : 1.f / l;
      const float lse_e = none ? -INFINITY : (m + log2f(l) - (Q8 ? kWeightLog2 : 0.f)) * 0.6931471805599453f;
      const int64_t row = (int64_t)(q0 + (valid ? tok : 0)) * p.Hq + hq;
      if (p.S > 1) {
        // this split's normalised partial (fp32) and its natural-log LSE
        float* orow = p.part_o + ((int64_t)split * p.part_rows + row) * D;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          uint32_t raw[2][32];
          tmem_ld32(lane_base + col_o + h * 64, raw[0]);
          tmem_ld32(lane_base + col_o + h * 64 + 32, raw[1]);
          tmem_wait_ld();
          if (valid) {
#pragma unroll
            for (int e = 0; e < 64; e += 4)
              *reinterpret_cast<float4*>(orow + h * 64 + e) =
                  make_float4(__uint_as_float(raw[e >> 5][e & 31]) * inv, __uint_as_float(raw[e >> 5][(e & 31) + 1]) * inv,
                              __uint_as_float(raw[e >> 5][(e & 31) + 2]) * inv,
                              __uint_as_float(raw[e >> 5][(e & 31) + 3]) * inv);
          }
        }
        if (valid) p.part_lse[(int64_t)split * p.part_rows + row] = lse_e;
      } else {
        const float sc = inv * (p.out_scale ? p.out_scale[hq] : 1.f);
        __nv_bfloat16* orow = p.out + (int64_t)(q0 + (valid ? tok : 0)) * p.out_stride_tok + (int64_t)hq * D;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          uint32_t raw[2][32];
          tmem_ld32(lane_base + col_o + h * 64, raw[0]);
          tmem_ld32(lane_base + col_o + h * 64 + 32, raw[1]);
          tmem_wait_ld();
          if (valid) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint32_t* r8 = &raw[c >> 2][(c & 3) * 8];
              uint4 v;
              v.x = pack_bf16(__uint_as_float(r8[0]) * sc, __uint_as_float(r8[1]) * sc);
              v.y = pack_bf16(__uint_as_float(r8[2]) * sc, __uint_as_float(r8[3]) * sc);
              v.z = pack_bf16(__uint_as_float(r8[4]) * sc, __uint_as_float(r8[5]) * sc);
              v.w = pack_bf16(__uint_as_float(r8[6]) * sc, __uint_as_float(r8[7]) * sc);
              if (staged)
                *reinterpret_cast<uint4*>(swarp + h * Cfg::Q_HALF + lane * 128 + ((c ^ (r & 7)) << 4)) = v;
              else
                *reinterpret_cast<uint4*>(orow + h * 64 + c * 8) = v;
            }
          }
          if (staged) {
            fence_proxy_async_smem();  // this lane's rows, visible to the copy
            __syncwarp();
            if (lane == 0)
              tma_store_3d(&tmo, swarp + h * Cfg::Q_HALF, h * 64, hk * GROUP,
                           q0 + t0 + t * TOK + (warp & 3) * (32 / GROUP));
          }
        }
        if (staged && lane == 0) {
          bulk_commit_group();
          bulk_wait_group_read0();  // shared memory is released when the CTA exits
        }
        if (valid && p.lse) p.lse[row] = lse_e;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMma) tmem_dealloc(tmem, 512);
}

template <int D, int GROUP, bool Q8, typename Stage>
int launch_prefill(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to,
                   const Stage& stage, const PrefillParams& prm, int max_q, cudaStream_t stream) {
  using Cfg = PrefillCfg<D>;
  constexpr int TOK = kTiles * kBM / GROUP;  // query tokens per CTA
  constexpr int smem = Q8 ? Cfg::SMEM_Q8 : Cfg::SMEM_BYTES;
  static bool attr_done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    if (cudaFuncSetAttribute(prefill_tcgen05_kernel<D, GROUP, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
        cudaSuccess)
      return LKV_ERR_CUDA;
    attr_done[dev] = true;
  }
  dim3 grid((max_q + TOK - 1) / TOK, prm.Hkv, prm.B * prm.S);
  prefill_tcgen05_kernel<D, GROUP, Q8><<<grid, kThreads, smem, stream>>>(tq, tk, tv, to, prm, stage);
  return cudaGetLastError() == cudaSuccess ? LKV_OK : LKV_ERR_CUDA;
}

}  // namespace

namespace {
// LKV_OK, or why the arguments are refused; *empty: there is nothing to do.
int check_args(const PrefillArgs& a, bool* empty) {
  *empty = false;
  if (a.head_dim != 64 && a.head_dim != 128) return LKV_ERR_UNSUPPORTED;
  if (a.num_kv_heads <= 0 || a.num_q_heads <= 0 || a.num_q_heads % a.num_kv_heads) return LKV_ERR_INVALID_ARGUMENT;
  const int group = a.num_q_heads / a.num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8) return LKV_ERR_UNSUPPORTED;
  if (a.batch < 0 || a.total_q < 0 || a.max_q < 0 || a.max_pages_per_seq < 0) return LKV_ERR_INVALID_ARGUMENT;
  if (a.batch == 0 || a.total_q == 0 || a.max_q == 0) {
    *empty = true;
    return LKV_OK;
  }
  const bool q8 = a.stage_k != nullptr;
  const bool pool = a.pool_k && a.pool_v && a.num_pages > 0;
  if (!a.q || (!pool && !q8) || (!a.block_table && a.max_pages_per_seq) || !a.seq_k || !a.cu_q || !a.out)
    return LKV_ERR_INVALID_ARGUMENT;
  if (q8 && (!a.stage_v || !a.q8_scales || a.stage_width < 1 || (int64_t)a.stage_width * a.batch >= INT32_MAX ||
             a.q8_pages < 0))
    return LKV_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(a.q) & 15) || ((a.q_stride_tok * 2) & 15)) return LKV_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(a.out) & 15) || ((a.out_stride_tok * 2) & 15)) return LKV_ERR_INVALID_ARGUMENT;
  if (a.batch > 65535 || a.num_kv_heads > 65535) return LKV_ERR_UNSUPPORTED;
  if (!a.error_word && !q8) return LKV_ERR_INVALID_ARGUMENT;
  const int S = a.kv_splits < 1 ? 1 : a.kv_splits;
  if (S > 1) {
    // key splits need a non-causal call (every query sees the same key range); with 8-bit pages, where the
    // older keys are most of a span's, causal ones take them too
    if ((a.causal && !q8) || S > kMaxKvSplits || (int64_t)a.batch * S > 65535) return LKV_ERR_UNSUPPORTED;
    if (!a.part_o || !a.part_lse || (reinterpret_cast<uintptr_t>(a.part_o) & 15)) return LKV_ERR_INVALID_ARGUMENT;
  }
  return LKV_OK;
}
}  // namespace

int prefill_paged_q8(const PrefillArgs& a, const void* codes, int staged) {
  bool empty;
  const int st = check_args(a, &empty);
  if (st != LKV_OK || empty) return st;
  if (!a.stage_k) return LKV_ERR_INVALID_ARGUMENT;
  if (staged == 0 && a.stage_width > a.max_pages_per_seq) return LKV_ERR_INVALID_ARGUMENT;
  if (staged == 0 || staged == 2) {
    const int rc = stage_pages(codes, a.q8_scales, a.q8_pages, a.block_table, a.block_table_stride, a.num_q8, a.seq_k,
                               a.batch, a.max_pages_per_seq, a.stage_k, a.stage_v, a.stage_width, a.num_kv_heads,
                               a.head_dim, a.error_word, static_cast<cudaStream_t>(a.stream));
    if (rc != LKV_OK) return rc;
  }
  return prefill_paged(a);
}

int prefill_paged(const PrefillArgs& a) {
  bool empty;
  int st = check_args(a, &empty);
  if (st != LKV_OK || empty) return st;
  const int group = a.num_q_heads / a.num_kv_heads, S = a.kv_splits < 1 ? 1 : a.kv_splits;
  const bool q8 = a.stage_k != nullptr, pool = a.pool_k && a.pool_v && a.num_pages > 0;

  CUtensorMap tq, tk, tv;
  st = make_query_tensor_map(&tq, a.q, a.total_q, a.q_stride_tok, a.num_q_heads, a.head_dim, group);
  if (st != LKV_OK) return st;
  StageMaps stage;
  if (q8) {
    const int64_t staged = (int64_t)a.stage_width * a.batch;
    st = make_pool_tensor_map(&stage.k, a.stage_k, staged, a.num_kv_heads, a.head_dim);
    if (st != LKV_OK) return st;
    st = make_pool_tensor_map(&stage.v, a.stage_v, staged, a.num_kv_heads, a.head_dim);
    if (st != LKV_OK) return st;
  }
  if (pool) {
    st = make_pool_tensor_map(&tk, a.pool_k, a.num_pages, a.num_kv_heads, a.head_dim);
    if (st != LKV_OK) return st;
    st = make_pool_tensor_map(&tv, a.pool_v, a.num_pages, a.num_kv_heads, a.head_dim);
    if (st != LKV_OK) return st;
  } else {  // no bf16 pages: keys past a row's end read as zeros past the stage
    tk = stage.k;
    tv = stage.v;
  }
  // The output has the query's [token][head][dim] geometry: full tiles are stored
  // a warp's 32 rows at a time (unused when the map cannot be built).
  CUtensorMap to;
  memset(&to, 0, sizeof(to));
  const int tma_out = S == 1 && make_query_tensor_map(&to, a.out, a.total_q, a.out_stride_tok, a.num_q_heads,
                                                      a.head_dim, group, 32) == LKV_OK;

  PrefillParams prm{};
  prm.bt = a.block_table;
  prm.bt_stride = a.block_table_stride;
  prm.seq_k = a.seq_k;
  prm.cu_q = a.cu_q;
  prm.out = static_cast<__nv_bfloat16*>(a.out);
  prm.out_stride_tok = a.out_stride_tok;
  prm.lse = a.lse;
  prm.out_scale = a.out_scale;
  prm.err = a.error_word;
  prm.B = a.batch;
  prm.Hq = a.num_q_heads;
  prm.Hkv = a.num_kv_heads;
  prm.W = a.max_pages_per_seq;
  // (ids past the map's end read as zeros)
  prm.num_pages = pool ? a.num_pages : (int64_t)a.stage_width * a.batch;
  prm.causal = a.causal ? 1 : 0;
  prm.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  prm.S = S;
  prm.part_o = a.part_o;
  prm.part_lse = a.part_lse;
  prm.part_rows = (int64_t)a.total_q * a.num_q_heads;
  prm.tma_out = tma_out;
  prm.num_q8 = a.num_q8;
  prm.q8_scales = a.q8_scales;
  prm.q8_pages = a.q8_pages;
  prm.stage_width = a.stage_width;
  prm.has_pool = pool;
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  int rc = LKV_OK;
#define LKV_PF(DD, GG)                                                                        \
  rc = q8 ? launch_prefill<DD, GG, true>(tq, tk, tv, to, stage, prm, a.max_q, stream)          \
          : launch_prefill<DD, GG, false>(tq, tk, tv, to, NoStageMaps{}, prm, a.max_q, stream); \
  break
  if (a.head_dim == 128) {
    switch (group) {
      case 1: LKV_PF(128, 1);
      case 2: LKV_PF(128, 2);
      case 4: LKV_PF(128, 4);
      default: LKV_PF(128, 8);
    }
  } else {
    switch (group) {
      case 1: LKV_PF(64, 1);
      case 2: LKV_PF(64, 2);
      case 4: LKV_PF(64, 4);
      default: LKV_PF(64, 8);
    }
  }
#undef LKV_PF
  if (rc != LKV_OK || S == 1) return rc;
  // exact LSE merge of the splits into out (x out_scale) and lse
  return merge_partials(a.part_o, a.part_lse, S, prm.part_rows, a.head_dim, a.num_q_heads,
                        prm.part_rows * a.head_dim, prm.part_rows, a.out_scale, a.out, a.lse, stream,
                        a.out_stride_tok, a.cu_q, a.batch);
}

// Key splits of a call over 8-bit pages, causal or not: what the waves of CTAs take, in blocks (about 1.5 us), with
// the start and end of a CTA as 2.5 of them, and the merge launch as as many, besides the partials' way through memory.
// Short spans gain from them, long ones lose (us at 1 / 2 / 3 / 4 / 6 / 8 splits): one row of 8 tokens over 8192 keys
// 105 / 61 / 46 / 38 / 31 / 27; four of 128 over 2048 42 / 35 / 29 / 27 / 34 / 33; two of 1024 over 8192 235 / 287 /
// 304 / 306 / 347 / 394.
int prefill_q8_split_plan(int batch, int max_q, int total_q, int num_q_heads, int num_kv_heads, int head_dim,
                          int max_pages, int* kv_splits) {
  if (!kv_splits) return LKV_ERR_INVALID_ARGUMENT;
  *kv_splits = 1;
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return LKV_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return LKV_ERR_UNSUPPORTED;
  if (batch <= 0 || max_q <= 0 || max_pages <= 0) return LKV_OK;
  const int group = num_q_heads / num_kv_heads;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return LKV_ERR_CUDA;
  const int64_t tok_per_cta = (int64_t)kTiles * kBM / group;
  const int64_t ctas = (max_q + tok_per_cta - 1) / tok_per_cta * num_kv_heads * batch;
  const int64_t blocks = ((int64_t)max_pages * kPageTok + kBN - 1) / kBN;
  const double split_us = 2.0 * total_q * num_q_heads * head_dim * 4 / 5e6;  // a partial written and read
  double best = 1e30;
  for (int s = 1; s <= kMaxKvSplits; ++s) {
    if (s > 1 && (s > blocks || (int64_t)batch * s > 65535)) break;
    const double waves = (double)((ctas * s + sms - 1) / sms);
    const double cost = waves * ((double)((blocks + s - 1) / s) + 2.5) + (s > 1 ? 2.5 + s * split_us / 1.5 : 0.0);
    if (cost < best - 1e-9) {
      best = cost;
      *kv_splits = s;
    }
  }
  return LKV_OK;
}

// Key splits for a non-causal call: with one CTA per SM, a grid of C CTAs runs
// ceil(C / SMs) waves of equal CTAs of `blocks` key blocks; splitting the keys S
// ways gives S * C CTAs of blocks / S, ceil(S * C / SMs) / S waves, plus per
// extra split the partials' write and merge and the extra CTAs' start-up, about
// 28 block-times (measured on the Wan-1.3B shape: 456 CTAs x 256 blocks ran
// 1.80 / 1.70 / 1.68 / 1.69 / 1.71 / 1.81 ms at S = 1 / 2 / 3 / 4 / 5 / 8).
// Short key ranges (under 16 blocks per split) are not split.
int prefill_split_plan(int batch, int max_q, int num_q_heads, int num_kv_heads, int head_dim, int max_pages,
                       int causal, int* kv_splits) {
  if (!kv_splits) return LKV_ERR_INVALID_ARGUMENT;
  *kv_splits = 1;
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return LKV_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return LKV_ERR_UNSUPPORTED;
  if (causal || batch <= 0 || max_q <= 0 || max_pages <= 0) return LKV_OK;
  const int group = num_q_heads / num_kv_heads;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return LKV_ERR_CUDA;
  const int64_t tok_per_cta = (int64_t)kTiles * kBM / group;
  const int64_t ctas = (max_q + tok_per_cta - 1) / tok_per_cta * num_kv_heads * batch;
  const int64_t blocks = ((int64_t)max_pages * kPageTok + kBN - 1) / kBN;
  double best = 1e30;
  for (int s = 1; s <= kMaxKvSplits; ++s) {
    if (s > 1 && (blocks / s < 16 || (int64_t)batch * s > 65535)) break;
    const double waves = (double)((ctas * s + sms - 1) / sms) / s;
    const double cost = waves * (double)blocks + 28.0 * (s - 1);
    if (cost < best - 1e-9) {
      best = cost;
      *kv_splits = s;
    }
  }
  return LKV_OK;
}

}  // namespace lkv
