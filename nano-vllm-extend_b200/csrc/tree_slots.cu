// Positions and cache slots of a batch's drafted nodes, from the sequences'
// lengths, trees and block tables, without a host round trip.
//
//   position[row] = context_len + depth of the node
//   slot[row]     = slot of logical position context_len + number of the node
//                   (where the node's key and value wait during the check), or,
//                   with accepted: of context_len + depth for the nodes on the
//                   accepted path and -1 for the others (where they belong for good)
//
// A few KB in and out: the call is as long as its launch and two dependent loads.
// One thread per row; a CTA keeps the parents of its rows and of the 63 rows on
// either side in shared memory (a tree has at most 64 rows), so the walks to the
// root stay on chip.  Every row is written, so rows behind the last sequence and
// those of a malformed one get position 0 and slot -1, which stores nothing.
#include "tree.cuh"

namespace gdn {

constexpr int kSlotThreads = 64;

__global__ void __launch_bounds__(kSlotThreads) tree_slot_kernel(
    const int32_t* __restrict__ tables, int64_t table_stride, int max_blocks,
    const int32_t* __restrict__ ctx, const int32_t* __restrict__ cu, int n_seqs,
    const int32_t* __restrict__ parents, const int32_t* __restrict__ accepted, int max_nodes,
    int block_size, int64_t n_rows, int64_t* __restrict__ pos_out, int32_t* __restrict__ slot_out,
    int32_t* status) {
  constexpr int HALO = kMaxTreeNodes - 1;
  __shared__ int s_par[kSlotThreads + 2 * HALO];
  const int64_t t0 = (int64_t)blockIdx.x * kSlotThreads;
  for (int i = threadIdx.x; i < kSlotThreads + 2 * HALO; i += kSlotThreads) {
    const int64_t t = t0 - HALO + i;
    s_par[i] = t >= 0 && t < n_rows ? parents[t] : -1;
  }
  if (blockIdx.x == 0) {            // malformed sequences are flagged even where no row finds them
    int64_t at;
    int m;
    for (int i = threadIdx.x; i < n_seqs; i += kSlotThreads)
      tree_rows(cu, i, n_rows, max_nodes, status, at, m);
  }
  int r = warp_seq_of(cu, n_seqs, t0 + (threadIdx.x & ~31));
  const int64_t t = t0 + threadIdx.x;
  while (r < n_seqs && (int64_t)cu[r + 1] <= t) ++r;
  int64_t start = 0;
  int n = 0, c = 0, last = -1;
  const bool mine = t < n_rows && r < n_seqs &&
                    tree_rows(cu, r, n_rows, max_nodes, status, start, n) && t >= start &&
                    t < start + n;
  if (mine) {
    c = ctx[r];
    if (accepted != nullptr) last = accepted[r];
  }
  __syncthreads();
  if (t >= n_rows) return;
  int64_t pos = 0, slot = -1;
  if (mine) {
    const int i = (int)(t - start);
    const int* par = s_par + (start - (t0 - HALO));   // par[j]: node j of this sequence
    int depth = 0, p = par[i];
    bool bad = c < 0, kept = true;
    for (int j = i; p != -1; ++depth) {               // p < j: the walk ends
      if (p < 0 || p >= j) {
        bad = true;
        break;
      }
      j = p;
      p = par[j];
    }
    if (accepted != nullptr) {
      bad |= last < -1 || last >= n;
      int j = bad ? -1 : last;
      while (j > i) {
        p = par[j];
        if (p < -1 || p >= j) {
          bad = true;
          break;
        }
        j = p;
      }
      kept = j == i;
    }
    if (bad) {
      if (status) atomicOr(status, c < 0 ? GDN_STATUS_BAD_SEQLEN : GDN_STATUS_BAD_TREE);
    } else {
      pos = (int64_t)c + depth;
      const unsigned at = (unsigned)c + (accepted != nullptr ? depth : i);
      if (kept) {
        const unsigned blk = at / (unsigned)block_size;
        const int64_t page = blk < (unsigned)max_blocks ? tables[r * table_stride + blk] : -1;
        slot = page * block_size + (at - blk * (unsigned)block_size);
        if (page < 0 || slot > INT32_MAX) {
          if (status) atomicOr(status, GDN_STATUS_BAD_SLOT);
          slot = -1;
        }
      }
    }
  }
  pos_out[t] = pos;
  slot_out[t] = (int32_t)slot;
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_tree_slot_map(const int32_t* block_tables, int64_t table_stride,
                                 int32_t max_blocks, const int32_t* context_lens,
                                 const int32_t* cu_seqlens, int32_t n_seqs,
                                 const int32_t* parents, const int32_t* accepted,
                                 int32_t max_nodes, int32_t block_size, int64_t n_rows,
                                 int64_t* positions, int32_t* slot_mapping, int32_t* status,
                                 void* stream) {
  clear_error();
  const char* fn = "gdn_tree_slot_map";
  GDN_REQUIRE(n_seqs >= 0 && n_rows >= 0 && max_nodes >= 0, "%s: bad sizes (n_seqs=%d, n_rows=%lld)",
              fn, n_seqs, (long long)n_rows);
  GDN_UNSUPPORTED(max_nodes <= kMaxTreeNodes, "%s: %d nodes in a tree (max %d)", fn, max_nodes,
                  kMaxTreeNodes);
  GDN_REQUIRE(block_size > 0 && max_blocks >= 0 && table_stride >= max_blocks,
              "%s: bad block tables (block_size=%d, max_blocks=%d, row stride %lld)", fn,
              block_size, max_blocks, (long long)table_stride);
  if (n_rows == 0) return GDN_OK;
  GDN_REQUIRE((block_tables || max_blocks == 0 || n_seqs == 0) && cu_seqlens && parents &&
                  positions && slot_mapping && (context_lens || n_seqs == 0),
              "%s: null pointer", fn);
  const int64_t ctas = (n_rows + kSlotThreads - 1) / kSlotThreads;
  GDN_UNSUPPORTED(ctas < (1ll << 31), "%s: too many rows", fn);
  tree_slot_kernel<<<(unsigned)ctas, kSlotThreads, 0, (cudaStream_t)stream>>>(
      block_tables, table_stride, max_blocks, context_lens, cu_seqlens, n_seqs, parents, accepted,
      max_nodes, block_size, n_rows, positions, slot_mapping, status);
  return check_launch(fn);
}
