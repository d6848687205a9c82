// Trees of drafted tokens, as every tree operator reads them.
//
// Sequence r owns rows [cu[r], cu[r+1]), one per node, parents before their
// children: parents[row] is the parent's number within the sequence, in
// [-1, own number), -1 for a node that hangs under the stored context.  A node
// sees the context, its ancestors and itself.
#pragma once

#include "common.cuh"

namespace gdn {

constexpr int kMaxTreeNodes = GDN_MAX_TREE_NODES;

// Rows of sequence r; false (and flagged) where cu_seqlens is malformed there
// or the sequence has more than max_nodes rows.
__device__ __forceinline__ bool tree_rows(const int32_t* __restrict__ cu, int r, int64_t n_tokens,
                                          int max_nodes, int32_t* status, int64_t& start, int& n) {
  start = cu[r];
  const int64_t len = (int64_t)cu[r + 1] - start;
  if (start < 0 || len < 0 || len > max_nodes || start + len > n_tokens) {
    if (status) atomicOr(status, GDN_STATUS_BAD_SEQLEN);
    return false;
  }
  n = (int)len;
  return true;
}

// Parent p of node i as given, or -1 (flagged) where it is not an earlier node:
// every walk towards the root therefore ends, and stays inside the sequence.
__device__ __forceinline__ int tree_parent(int p, int i, int32_t* status) {
  if (p >= -1 && p < i) return p;
  if (status) atomicOr(status, GDN_STATUS_BAD_TREE);
  return -1;
}

// Sequence of flat row t for a whole warp: the number of sequences that end at
// or before t (empty ones are passed over); n_seqs for a row behind the last.
__device__ __forceinline__ int warp_seq_of(const int32_t* __restrict__ cu, int n_seqs, int64_t t) {
  int c = 0;
  for (int i = 1 + (threadIdx.x & 31); i <= n_seqs; i += 32) c += (int64_t)cu[i] <= t;
  return __reduce_add_sync(0xffffffffu, c);
}

}  // namespace gdn
