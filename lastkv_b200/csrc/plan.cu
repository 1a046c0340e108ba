// A step's block tables, slot maps, positions and boundary commits from request lengths,
// in one launch (sm_100a): the device form of the host plan of the merged pool
// (vllm/src/lastkv/vllm/backends/rmarin_flashinfer/fastpath.py:373-454), for steps that
// are captured in a CUDA graph and advance without the host.
//
// For row b with p0 computed tokens, n new ones and session slot s (C the chunk, P = 16,
// RP = 2C / P ring pages per slot):
//   last = p0 + n - 1, cur = floor(last / C) C, rec = max(0, cur - C), ns = rec / P,
//   np = ceil((last + 1 - rec) / P)
//   table[l, b, j] = src_table[s, j]                                    j < ns
//                  = ring_base[l] + s RP + (ns % RP + j - ns) % RP      ns <= j < ns + np
//                  = ring_base[l]                                       beyond
//   seq_k[b] = last + 1;  token p of the row: position p, ring slot s 2C + p % 2C,
//   shared slot src_table[s, p / P] P + p % P
//   a commit of chunk [p0 - C, p0) where n > 0, p0 > 0 and p0 % C = 0: the step is the
//   first after that chunk (spans never cross a boundary, so each chunk gets exactly one)
// A row with slot < 0 is padding: one token on the scratch pages.  A row that breaks the
// plan's rules (a span over a chunk boundary, past the capacity, a slot that is not
// there, n < 1, more tokens than the buffers hold) is recorded in the error word and runs
// on the scratch pages too: it reads no other page, however long, and commits nothing.
//
// Writing L x B x W table words is the floor.  grid = (rows + 1) x parts x layer runs: a
// block takes one part of a row's columns (four neighbours per thread where the width allows
// 16-byte stores), computes each once and stores it for its run of layers; few rows and
// columns get more runs, so that the GPU is filled.  32 layers, chunks of 1024, tables of 512
// columns: 8 decode rows 4.0 us (one run of layers 5.7), 64 rows 5.2 us (4-byte stores 6.5);
// 64 spans in tables of 8192 columns 16.2 us, 4.2 TB/s of stores (4-byte stores 22.3).  The extra row fills the unused tokens
// and commit rows.  Every block scans the rows' lengths itself (a few KB from L2), which
// costs less than a second launch.

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.cuh"

namespace lkv {

namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanKernelId = 12;

struct Row {
  int p0, n, slot;  // slot < 0: padding, runs on the scratch pages
  int tokens;       // token slots that the row takes in the buffers
  bool bad;
};

__device__ __forceinline__ Row load_row(const PlanArgs& a, int b) {
  Row r;
  r.p0 = a.num_computed[b];
  r.n = a.num_new[b];
  r.slot = a.slots[b];
  r.bad = false;
  if (r.slot < 0) {
    r.p0 = 0;
    r.n = 1;
  } else {
    const int64_t end = (int64_t)r.p0 + r.n;
    r.bad = r.slot >= a.num_slots || r.p0 < 0 || r.n < 1 || r.n > a.max_tokens || end > a.max_sequence_tokens ||
            r.p0 / a.chunk != (int)((end - 1) / a.chunk);
  }
  r.tokens = max(0, min(r.n, a.max_tokens));
  return r;
}

__device__ __forceinline__ bool row_commits(const PlanArgs& a, const Row& r) {
  return !r.bad && r.slot >= 0 && r.p0 > 0 && r.p0 % a.chunk == 0;
}

template <int VEC>
__global__ void __launch_bounds__(kPlanThreads) plan_step_kernel(const PlanArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, part = blockIdx.y, parts = gridDim.y;
  const bool tail = b == a.batch, once = blockIdx.z == 0;  // what a row has once: by the first layer run
  const int l0 = (int)((int64_t)a.num_layers * blockIdx.z / gridDim.z);
  const int l1 = (int)((int64_t)a.num_layers * (blockIdx.z + 1) / gridDim.z);
  if (tail && !once) return;
  // tokens and commits of the rows before this one, and of all rows (saturating: a sum
  // past the buffers is past them)
  __shared__ int64_t s_tok[2][kPlanThreads / 32];
  __shared__ int s_com[2][kPlanThreads / 32];
  int64_t tok[2] = {0, 0};
  int com[2] = {0, 0};
  for (int i = threadIdx.x; i < a.batch; i += kPlanThreads) {
    const Row r = load_row(a, i);
    const int c = row_commits(a, r) ? 1 : 0;
    tok[1] += r.tokens;
    com[1] += c;
    if (i < b) {
      tok[0] += r.tokens;
      com[0] += c;
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      tok[k] += __shfl_xor_sync(0xffffffffu, tok[k], o);
      com[k] += __shfl_xor_sync(0xffffffffu, com[k], o);
    }
    if ((threadIdx.x & 31) == 0) {
      s_tok[k][threadIdx.x >> 5] = tok[k];
      s_com[k][threadIdx.x >> 5] = com[k];
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    tok[k] = 0;
    com[k] = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      tok[k] += s_tok[k][w];
      com[k] += s_com[k][w];
    }
  }
  // A row that does not fit the buffers runs on the scratch pages and comes again in another step,
  // which commits its chunk: not this one (a commit blends in place).  After the first such row
  // none fits.
  int fits = a.batch;
  if (tok[1] > a.max_tokens) {
    __shared__ int s_fits[3];
    if (threadIdx.x == 0) {
      int64_t sum = 0;
      int i = 0, before = 0, listed = 0;
      for (; i < a.batch; ++i) {
        const Row r = load_row(a, i);
        sum += r.tokens;
        if (sum > a.max_tokens) break;
        const int c = row_commits(a, r) ? 1 : 0;
        listed += c;
        before += i < b ? c : 0;
      }
      s_fits[0] = i;
      s_fits[1] = before;
      s_fits[2] = listed;
    }
    __syncthreads();
    fits = s_fits[0];
    com[0] = s_fits[1];
    com[1] = s_fits[2];
  }
  const int64_t first_tok = tok[0] < a.max_tokens ? tok[0] : a.max_tokens;
  const int64_t all_tok = tok[1] < a.max_tokens ? tok[1] : a.max_tokens;
  const int ppc = a.chunk / LKV_PAGE_SIZE, ring_pages = 2 * ppc;
  const int gtid = part * kPlanThreads + threadIdx.x, gsize = parts * kPlanThreads;
  const int64_t pad_ring = (int64_t)a.scratch_ring_page * LKV_PAGE_SIZE;
  const int64_t pad_src = (int64_t)a.scratch_src_page * LKV_PAGE_SIZE;

  if (tail) {
    for (int64_t t = all_tok + gtid; t < a.max_tokens; t += gsize) {
      a.positions[t] = 0;
      a.ring_slots[t] = pad_ring;
      a.src_slots[t] = pad_src;
    }
    for (int64_t i = (int64_t)com[1] * ppc + gtid; i < (int64_t)a.batch * ppc; i += gsize) {
      a.commit_raw[i] = 0;
      a.commit_ring[i] = 0;
    }
    if (gtid == 0) {
      a.cu_q[a.batch] = (int)all_tok;
      a.commit_count[0] = com[1];
    }
    return;
  }

  const Row r = load_row(a, b);
  const bool over = b >= fits;
  const bool real = r.slot >= 0 && !r.bad && !over;
  // a row on the scratch pages is as long as its tokens, every page of it the scratch page
  const int len = real ? r.p0 + r.n : max(1, (int)(min(first_tok + r.tokens, (int64_t)a.max_tokens) - first_tok));
  const int scratch = real ? 0 : (len - 1) / LKV_PAGE_SIZE + 1;
  if (once && gtid == 0) {
    if (r.bad || over) report_error(a.error_word, DEVERR_BAD_SPAN, kPlanKernelId, b);
    a.cu_q[b] = (int)first_tok;
    a.seq_k[b] = len;
  }
  const int last = r.p0 + r.n - 1;
  const int rec = max(0, last / a.chunk * a.chunk - a.chunk);
  const int ns = real ? rec / LKV_PAGE_SIZE : 0;
  const int np = real ? (last - rec) / LKV_PAGE_SIZE + 1 : 0;  // (last + 16 may pass 2^31)
  const int32_t* src = a.src_table + (int64_t)(real ? r.slot : 0) * a.src_table_stride;
  const int64_t layer = (int64_t)a.batch * a.width;
  for (int j0 = gtid * VEC; j0 < a.width; j0 += gsize * VEC) {
    int v[VEC];
    int ring = j0 < ns + np ? (ns % ring_pages + max(j0 - ns, 0)) % ring_pages : 0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int j = j0 + e;
      v[e] = 0;
      if (j < ns) {
        v[e] = src[j];
      } else if (j < ns + np) {
        v[e] = r.slot * ring_pages + ring;
        if (++ring == ring_pages) ring = 0;
      } else if (j < scratch) {
        v[e] = a.scratch_ring_page;
      }
    }
    int32_t* dst = a.block_tables + (int64_t)b * a.width + j0;
    for (int l = l0; l < l1; ++l) {
      const int base = a.ring_base[l];
      if constexpr (VEC == 4) {
        *reinterpret_cast<int4*>(dst + l * layer) =
            make_int4(j0 < ns ? v[0] : v[0] + base, j0 + 1 < ns ? v[1] : v[1] + base,
                      j0 + 2 < ns ? v[2] : v[2] + base, j0 + 3 < ns ? v[3] : v[3] + base);
      } else {
        dst[l * layer] = j0 < ns ? v[0] : v[0] + base;
      }
    }
  }
  if (!once) return;
  for (int i = gtid; i < r.tokens; i += gsize) {
    const int64_t t = first_tok + i;
    if (t >= a.max_tokens) break;
    const int p = r.p0 + i;
    a.positions[t] = real ? p : 0;
    a.ring_slots[t] = real ? (int64_t)r.slot * 2 * a.chunk + p % (2 * a.chunk) : pad_ring;
    a.src_slots[t] = real ? (int64_t)src[p / LKV_PAGE_SIZE] * LKV_PAGE_SIZE + p % LKV_PAGE_SIZE : pad_src;
  }
  if (!over && row_commits(a, r)) {
    const int page = (r.p0 - a.chunk) / LKV_PAGE_SIZE;
    const int32_t* own = a.src_table + (int64_t)r.slot * a.src_table_stride;
    for (int i = gtid; i < ppc; i += gsize) {
      a.commit_raw[(int64_t)com[0] * ppc + i] = own[page + i];
      a.commit_ring[(int64_t)com[0] * ppc + i] = a.ring_base[0] + r.slot * ring_pages + page % ring_pages + i;
    }
  }
}

}  // namespace

int plan_step(const PlanArgs& a, cudaStream_t stream) {
  if (a.batch < 0 || a.max_tokens < 0 || a.num_layers < 1 || a.num_slots < 1 || a.max_sequence_tokens < 1 ||
      a.chunk < LKV_PAGE_SIZE || a.chunk % LKV_PAGE_SIZE || a.chunk > (1 << 29))
    return LKV_ERR_INVALID_ARGUMENT;
  const int pages = (int)(((int64_t)a.max_sequence_tokens + LKV_PAGE_SIZE - 1) / LKV_PAGE_SIZE);
  // a row uses ceil((last + 1) / 16) columns: older pages and ring pages together
  if ((a.num_slots > 1 && a.src_table_stride < pages) || a.width < pages) return LKV_ERR_INVALID_ARGUMENT;
  if (a.batch == 0) return LKV_OK;
  if (!a.num_computed || !a.num_new || !a.slots || !a.src_table || !a.ring_base || !a.block_tables || !a.seq_k ||
      !a.cu_q || !a.positions || !a.ring_slots || !a.src_slots || !a.commit_raw || !a.commit_ring ||
      !a.commit_count)
    return LKV_ERR_INVALID_ARGUMENT;
  const bool wide = a.width % 4 == 0 && (reinterpret_cast<uintptr_t>(a.block_tables) & 15) == 0;
  const int per_block = kPlanThreads * (wide ? 4 : 1);
  const int parts = std::max(1, std::min((a.width + per_block - 1) / per_block, 65535));
  // two blocks per SM, if the layers allow
  const int64_t blocks = ((int64_t)a.batch + 1) * parts;
  const int runs = (int)std::min<int64_t>(std::min(a.num_layers, 65535), std::max<int64_t>(1, 2 * 148 / blocks));
  return launch_pdl(wide ? plan_step_kernel<4> : plan_step_kernel<1>,
                    dim3((unsigned)a.batch + 1, (unsigned)parts, (unsigned)runs), dim3(kPlanThreads), 0, stream,
                    a) == cudaSuccess
             ? LKV_OK
             : LKV_ERR_CUDA;
}

}  // namespace lkv
