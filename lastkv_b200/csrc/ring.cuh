// Book-keeping of a ring of DEPTH shared-memory slots that copies fill and one warp reads in
// order: which slot a step uses, the parity its barrier is waited on with, and how many copies
// are in flight.  Block j lies in slot j % DEPTH; its copy completes phase j / DEPTH there.
// Plain C++ where it is not compiled by nvcc.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LKV_RING_FN __host__ __device__ __forceinline__
#else
#define LKV_RING_FN inline
#endif

namespace lkv {

template <int DEPTH>
struct Ring {
  int slot = 0;        // of the oldest block that has not been read
  uint32_t phase = 0;  // its barrier's parity
  int flying = 0;      // copies issued and not read: they lie in slot, slot + 1, ...

  // The slot that the next copy goes to; flying < DEPTH.
  LKV_RING_FN int fill() {
    const int s = slot + flying;
    ++flying;
    return s < DEPTH ? s : s - DEPTH;
  }
  // The oldest block has been read (or waited for): its slot is free.
  LKV_RING_FN void next() {
    --flying;
    if (++slot == DEPTH) {
      slot = 0;
      phase ^= 1;
    }
  }
};

}  // namespace lkv
