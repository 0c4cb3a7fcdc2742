// Device helpers the 8-bit KV cache's kernels share.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace onpu_b200 {

// The rows of sequence b: cache rows pos .. pos + cnt - 1. False (and bit 32 of *err) where they are not
// all inside the cache of S rows or cnt is not in [0, T]; the sequence is then skipped.
__device__ __forceinline__ bool kv8_rows(const Kv8Rows &r, int b, int S, int &pos, int &cnt) {
    pos = r.pos[b];
    cnt = r.cnt ? r.cnt[b] : r.T;
    if (cnt >= 0 && cnt <= r.T && pos >= 0 && pos <= S - cnt) return true;
    atomicOr(r.err, 32);
    return false;
}

}  // namespace onpu_b200
