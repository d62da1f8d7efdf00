// What the attention kernels share: which keys a query row sees.
#pragma once

#include <climits>

#include "token_ops.h"

namespace illumina {
namespace gpu {

// Sequence n of a batch: q_len queries and k_len keys, the last query at the
// last key. Without a causal block a query sees all k_len keys; with one it
// stands at key position i + k_len - q_len and sees the keys of its own block
// of `block` keys and of the blocks before it.
struct AttnMask {
  int q_len, k_len, off, block;
  __device__ __forceinline__ AttnMask(const AttnParams &p, int n) {
    q_len = p.q_lens ? min(max(p.q_lens[n], 0), p.q_tokens) : p.q_tokens;
    k_len = p.k_lens ? min(max(p.k_lens[n], 0), p.k_tokens) : p.k_tokens;
    off = k_len - q_len;
    block = p.causal_block;
  }
  // Keys [0, end) are seen by row i; 0 for padding rows. Grows with i.
  __device__ __forceinline__ int key_end(int i) const {
    if (i >= q_len) return 0;
    if (!block) return k_len;
    const int at = i + off;
    if (at < 0) return 0;
    const long long end = ((long long)(at / block) + 1) * block;
    return end < k_len ? (int)end : k_len;
  }
  // First row that sees key j (j < k_len); q_len if none does.
  __device__ __forceinline__ int row_begin(int j) const {
    if (!block) return 0;
    const long long i = (long long)(j / block) * block - off;
    return i <= 0 ? 0 : i < q_len ? (int)i : q_len;
  }
};

}  // namespace gpu
}  // namespace illumina
