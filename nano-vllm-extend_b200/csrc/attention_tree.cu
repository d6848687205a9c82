// Attention of drafted nodes over a paged cache: node i of sequence r sees the
// cache's positions [0, context_len) and, at context_len + j, the nodes j on its
// path (itself included), whose keys and values already stand in the cache.  One
// node per sequence is the plain decode step, a chain the causal one.
//
//   o_i = sum_p softmax_p(scale q_i.k_p) v_p
//
// HBM: every cached key and value of a sequence is read once (4 D bytes per
// position and kv-head), so the G = HQ / HKV query heads of a kv-head and all
// nodes form the rows of one tile: 16 WM rows per CTA.  Work is split along the
// positions in chunks, so few sequences still fill the GPU and long ones do not
// run behind the others; with more than one chunk each writes its rows' running
// maximum, sum and weighted values in fp32 and a second launch joins them.
//
// One pass over a chunk with the running maximum and sum of the softmax: tiles
// of BN positions arrive by cp.async, three stages deep, rows swizzled for
// ldmatrix; WM warps over rows x WN warps over positions, scores and
// probabilities stay in registers (the score tile's accumulators are the next
// product's A operand).  Sums and statistics are fp32; the probabilities are
// rounded to bf16 as an operand of the second product, as the values are bf16.
//
// Positions behind the last node are filled with zeros, not read.  A node's
// value row that is not finite must not reach nodes off its path (probability
// zero times NaN): in tiles that hold nodes such rows are zeroed in shared
// memory and the nodes that do see them get NaN outputs.
#include "mma_util.cuh"
#include "tc_util.cuh"
#include "tree.cuh"

namespace gdn {

constexpr int kAttnStages = 3;

struct AttnArgs {
  const bf16* q;
  int64_t qs;
  const bf16 *k_cache, *v_cache;
  int64_t block_stride, token_stride, head_stride, num_blocks;
  int block_size;
  const int32_t* tables;
  int64_t table_stride;
  int max_blocks;
  const int32_t* ctx;
  const int32_t* cu;
  int n_seqs;
  const int32_t* parents;
  int max_nodes;
  int64_t n_tokens;
  int max_len;
  bf16* out;
  int HQ, HKV;
  float scale_log2;
  int chunk, chunks, row_tiles;   // positions per chunk, chunks of the longest sequence
  float* part_o;                  // [chunks][n_tokens * HQ][D]
  float2* part_ml;                // [chunks][n_tokens * HQ]: maximum (base 2), sum
  int32_t* status;
};

// Context length of sequence r; false (and flagged) where it is negative or the
// sequence is longer than the host's bound.
__device__ __forceinline__ bool attn_len(const AttnArgs& a, int r, int n, int64_t& c) {
  c = a.ctx[r];
  if (c < 0 || c + n > a.max_len) {
    if (a.status) atomicOr(a.status, GDN_STATUS_BAD_SEQLEN);
    return false;
  }
  return true;
}

template <int D, int WM, int WN, int BN>
struct AttnSmem {
  bf16 q[16 * WM][D];
  bf16 k[kAttnStages][BN][D];
  bf16 v[kAttnStages][BN][D];
  unsigned long long anc[kMaxTreeNodes];
  unsigned long long bad;
  int par[kMaxTreeNodes];
};

// Byte offset of 16-byte piece c of row r in a tile of D-wide bf16 rows: pieces
// of 8 consecutive rows land in different banks.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)(r * D * 2 + ((c ^ (r & 7)) << 4));
}

template <int D, int WM, int WN, int BN>
__global__ void __launch_bounds__(32 * WM * WN) attention_tree_kernel(const AttnArgs a) {
  using S = AttnSmem<D, WM, WN, BN>;
  constexpr int NT = 32 * WM * WN, BM = 16 * WM, PC = D / 8;
  constexpr int WT = BN / WN;                 // positions of a tile per warp
  static_assert(WT % 16 == 0, "a warp takes whole 16-position blocks");
  extern __shared__ __align__(128) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  int* pages = reinterpret_cast<int*>(smem_raw + sizeof(S));

  const int rt = blockIdx.x % a.row_tiles;
  const int kvh = (blockIdx.x / a.row_tiles) % a.HKV;
  const int seq = blockIdx.x / (a.row_tiles * a.HKV);
  const int chunk = blockIdx.y;
  const int G = a.HQ / a.HKV;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int wm = warp / WN, wn = warp - wm * WN;
  int64_t start, ctx;
  int n;
  if (!tree_rows(a.cu, seq, a.n_tokens, a.max_nodes, a.status, start, n) ||
      !attn_len(a, seq, n, ctx))
    return;
  const int row0 = rt * BM, rows = n * G;     // rows: node * G + head within the group
  const int total = (int)ctx + n;
  const int p_begin = chunk * a.chunk, p_end = min(total, p_begin + a.chunk);
  if (row0 >= rows || p_begin >= p_end) return;

  // the chunk's pages
  const int page0 = p_begin / a.block_size, n_pages = (p_end - 1) / a.block_size - page0 + 1;
  for (int i = tid; i < n_pages; i += NT) {
    int p = page0 + i < a.max_blocks ? a.tables[seq * a.table_stride + page0 + i] : -1;
    if (p < 0 || p >= a.num_blocks) {
      if (a.status) atomicOr(a.status, GDN_STATUS_BAD_SLOT);
      p = -1;
    }
    pages[i] = p;
  }
  if (tid < n) sm.par[tid] = tree_parent(a.parents[start + tid], tid, a.status);
  if (tid == 0) sm.bad = 0;
  // query rows
  for (int i = tid; i < BM * PC; i += NT) {
    const int r = i / PC, c = i - r * PC;
    const int row = row0 + r;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (row < rows) {
      const int node = row / G;
      u = *reinterpret_cast<const uint4*>(a.q + (start + node) * a.qs +
                                          (int64_t)(kvh * G + row - node * G) * D + c * 8);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(sm.q) + tile_at<D>(r, c)) = u;
  }
  __syncthreads();
  if (tid < n) {
    unsigned long long m = 0;
    for (int j = tid; j >= 0; j = sm.par[j]) m |= 1ull << j;
    sm.anc[tid] = m;
  }

  const int tiles = (p_end - p_begin + BN - 1) / BN;
  auto load_tile = [&](int tile, int stage) {
    const uint32_t k0 = tc::smem_u32(&sm.k[stage][0][0]), v0 = tc::smem_u32(&sm.v[stage][0][0]);
    for (int i = tid; i < BN * PC; i += NT) {
      const int r = i / PC, c = i - r * PC;
      const int p = p_begin + tile * BN + r;
      int64_t off = 0;
      uint32_t bytes = 0;
      if (p < p_end) {
        const int blk = p / a.block_size;
        const int page = pages[blk - page0];
        if (page >= 0) {
          off = page * a.block_stride + (p - blk * a.block_size) * a.token_stride +
                kvh * a.head_stride + c * 8;
          bytes = 16;
        }
      }
      tc::cp_async16(k0 + tile_at<D>(r, c), a.k_cache + off, bytes);
      tc::cp_async16(v0 + tile_at<D>(r, c), a.v_cache + off, bytes);
    }
  };
#pragma unroll
  for (int s = 0; s < kAttnStages - 1; ++s) {
    if (s < tiles) load_tile(s, s);
    tc::cp_async_commit();
  }

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
  const int my_row[2] = {row0 + wm * 16 + gr, row0 + wm * 16 + gr + 8};
  const uint32_t q_base = tc::smem_u32(&sm.q[0][0]);

  for (int tile = 0; tile < tiles; ++tile) {
    tc::cp_async_wait<kAttnStages - 2>();
    __syncthreads();                          // tile has arrived; the stage loaded next is free
    if (tile + kAttnStages - 1 < tiles)
      load_tile(tile + kAttnStages - 1, (tile + kAttnStages - 1) % kAttnStages);
    tc::cp_async_commit();
    const int stage = tile % kAttnStages;
    const int p_tile = p_begin + tile * BN;
    const bool edge = p_tile + BN > (int)ctx;   // holds nodes or positions behind them
    if (edge) {
      // value rows of nodes: zero what is not finite and note whose it is
      unsigned char* vt = reinterpret_cast<unsigned char*>(&sm.v[stage][0][0]);
      for (int i = tid; i < BN * PC; i += NT) {
        const int r = i / PC, c = i - r * PC;
        const int j = p_tile + r - (int)ctx;
        if (j < 0 || j >= n) continue;
        uint4* p = reinterpret_cast<uint4*>(vt + tile_at<D>(r, c));
        const uint4 u = *p;
        float f[8];
        unpack8(u, f);
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) finite &= fabsf(f[e]) <= 3.4e38f;
        if (!finite) {
          *p = make_uint4(0, 0, 0, 0);
          atomicOr(&sm.bad, 1ull << j);
        }
      }
      __syncthreads();
    }

    // scores of this warp's 16 rows x WT positions
    float s[WT / 8][4];
#pragma unroll
    for (int i = 0; i < WT / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
    const uint32_t k_base = tc::smem_u32(&sm.k[stage][0][0]);
#pragma unroll
    for (int kb = 0; kb < D / 16; ++kb) {
      uint32_t qa[4];
      mm::ldsm4(qa, q_base + tile_at<D>(wm * 16 + (lane & 15), kb * 2 + (lane >> 4)));
#pragma unroll
      for (int i = 0; i < WT / 8; i += 2) {
        uint32_t b[4];
        mm::ldsm4(b, k_base + tile_at<D>(wn * WT + i * 8 + (lane >> 4) * 8 + (lane & 7),
                                         kb * 2 + ((lane >> 3) & 1)));
        mm::mma16816(s[i], qa, b[0], b[1]);
        mm::mma16816(s[i + 1], qa, b[2], b[3]);
      }
    }
    // masks and scale
    if (edge || p_tile + BN > p_end) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const unsigned long long m = my_row[hh] < rows ? sm.anc[my_row[hh] / G] : 0ull;
#pragma unroll
        for (int i = 0; i < WT / 8; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int p = p_tile + wn * WT + i * 8 + 2 * tq + e;
            const int j = p - (int)ctx;
            const bool seen = p < p_end && (j < 0 || (j < n && (m >> (j & 63) & 1)));
            float& x = s[i][hh * 2 + e];
            x = seen ? x * a.scale_log2 : -INFINITY;
          }
      }
    } else {
#pragma unroll
      for (int i = 0; i < WT / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] *= a.scale_log2;
    }
    // running maximum and sum (base 2)
    uint32_t pa[WT / 16][4];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      float m = mx[hh];
#pragma unroll
      for (int i = 0; i < WT / 8; ++i) m = fmaxf(m, fmaxf(s[i][hh * 2], s[i][hh * 2 + 1]));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const float base = m == -INFINITY ? 0.f : m;    // a row that has seen nothing yet
      const float corr = exp2f(mx[hh] - base);
      mx[hh] = m;
      float add = 0.f;
#pragma unroll
      for (int i = 0; i < WT / 8; ++i) {
        s[i][hh * 2] = exp2f(s[i][hh * 2] - base);
        s[i][hh * 2 + 1] = exp2f(s[i][hh * 2 + 1] - base);
        add += s[i][hh * 2] + s[i][hh * 2 + 1];
      }
      sum[hh] = sum[hh] * corr + add;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][hh * 2] *= corr;
        o[i][hh * 2 + 1] *= corr;
      }
    }
#pragma unroll
    for (int i = 0; i < WT / 16; ++i) {
      pa[i][0] = mm::pack2(s[2 * i][0], s[2 * i][1]);
      pa[i][1] = mm::pack2(s[2 * i][2], s[2 * i][3]);
      pa[i][2] = mm::pack2(s[2 * i + 1][0], s[2 * i + 1][1]);
      pa[i][3] = mm::pack2(s[2 * i + 1][2], s[2 * i + 1][3]);
    }
    const uint32_t v_base = tc::smem_u32(&sm.v[stage][0][0]);
#pragma unroll
    for (int i = 0; i < WT / 16; ++i)
#pragma unroll
      for (int c = 0; c < D / 8; c += 2) {
        uint32_t b[4];
        mm::ldsm4t(b, v_base + tile_at<D>(wn * WT + i * 16 + (lane & 15), c + (lane >> 4)));
        mm::mma16816(o[c], pa[i], b[0], b[1]);
        mm::mma16816(o[c + 1], pa[i], b[2], b[3]);
      }
  }
  tc::cp_async_wait<0>();
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    sum[hh] += __shfl_xor_sync(0xffffffffu, sum[hh], 1);
    sum[hh] += __shfl_xor_sync(0xffffffffu, sum[hh], 2);
  }

  // join the WN warps of a row tile through shared memory (the stages are free)
  if constexpr (WN > 1) {
    __syncthreads();
    float2* ml = reinterpret_cast<float2*>(&sm.k[0][0][0]);          // [WN][BM]
    float* os = reinterpret_cast<float*>(ml + WN * BM);              // [WN][BM][D + 4]
    static_assert(sizeof(float2) * WN * BM + sizeof(float) * WN * BM * (D + 4) <=
                      sizeof(sm.k) + sizeof(sm.v),
                  "the joined rows fit the stages");
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = wm * 16 + gr + hh * 8;
      if (tq == 0) ml[wn * BM + r] = make_float2(mx[hh], sum[hh]);
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<float2*>(&os[(wn * BM + r) * (D + 4) + i * 8 + 2 * tq]) =
            make_float2(o[i][hh * 2], o[i][hh * 2 + 1]);
    }
    __syncthreads();
    // every thread finishes pieces of 4 columns
    for (int i = tid; i < BM * (D / 4); i += NT) {
      const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
      const int row = row0 + r;
      if (row >= rows) continue;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < WN; ++w) m = fmaxf(m, ml[w * BM + r].x);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WN; ++w) {
        const float2 p = ml[w * BM + r];
        const float f = exp2f(p.x - base);
        const float4 t = *reinterpret_cast<const float4*>(&os[(w * BM + r) * (D + 4) + c]);
        l = fmaf(p.y, f, l);
        acc.x = fmaf(t.x, f, acc.x);
        acc.y = fmaf(t.y, f, acc.y);
        acc.z = fmaf(t.z, f, acc.z);
        acc.w = fmaf(t.w, f, acc.w);
      }
      const int node = row / G;
      if (sm.anc[node] & sm.bad) acc.x = acc.y = acc.z = acc.w = __int_as_float(0x7fffffff);
      const int64_t at = (start + node) * a.HQ + kvh * G + row - node * G;
      if (a.chunks == 1) {
        const float inv = 1.f / l;
        uint2 u;
        u.x = mm::pack2(acc.x * inv, acc.y * inv);
        u.y = mm::pack2(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(a.out + at * D + c) = u;
      } else {
        const int64_t pr = chunk * (a.n_tokens * a.HQ) + at;
        *reinterpret_cast<float4*>(a.part_o + pr * D + c) = acc;
        if (c == 0) a.part_ml[pr] = make_float2(m, l);
      }
    }
  } else {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int row = my_row[hh];
      if (row >= rows) continue;
      const int node = row / G;
      const int64_t at = (start + node) * a.HQ + kvh * G + row - node * G;
      const bool nan = (sm.anc[node] & sm.bad) != 0;
      const int64_t pr = chunk * (a.n_tokens * a.HQ) + at;
      const float inv = a.chunks == 1 ? 1.f / sum[hh] : 1.f;
      if (a.chunks > 1 && tq == 0) a.part_ml[pr] = make_float2(mx[hh], sum[hh]);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        float x = o[i][hh * 2] * inv, y = o[i][hh * 2 + 1] * inv;
        if (nan) x = y = __int_as_float(0x7fffffff);
        if (a.chunks == 1)
          *reinterpret_cast<uint32_t*>(a.out + at * D + i * 8 + 2 * tq) = mm::pack2(x, y);
        else
          *reinterpret_cast<float2*>(a.part_o + pr * D + i * 8 + 2 * tq) = make_float2(x, y);
      }
    }
  }
}

// Joins a row's chunks: D / 4 lanes per (node, query head).
template <int D>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnArgs a) {
  constexpr int LPR = D / 4;
  const int seq = blockIdx.y;
  int64_t start, ctx;
  int n;
  if (!tree_rows(a.cu, seq, a.n_tokens, a.max_nodes, nullptr, start, n)) return;
  const int item = (int)(blockIdx.x * 256 + threadIdx.x);
  const int r = item / LPR, c = (item - r * LPR) * 4;
  if (r >= n * a.HQ) return;
  ctx = a.ctx[seq];
  if (ctx < 0 || ctx + n > a.max_len) return;
  const int chunks = (int)((ctx + n + a.chunk - 1) / a.chunk);
  const int64_t at = start * a.HQ + r, step = a.n_tokens * a.HQ;
  float m = -INFINITY;
  for (int i = 0; i < chunks; ++i) m = fmaxf(m, a.part_ml[i * step + at].x);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < chunks; ++i) {
    const float2 p = a.part_ml[i * step + at];
    const float f = exp2f(p.x - base);
    const float4 t = *reinterpret_cast<const float4*>(a.part_o + (i * step + at) * D + c);
    l = fmaf(p.y, f, l);
    acc.x = fmaf(t.x, f, acc.x);
    acc.y = fmaf(t.y, f, acc.y);
    acc.z = fmaf(t.z, f, acc.z);
    acc.w = fmaf(t.w, f, acc.w);
  }
  const float inv = 1.f / l;
  uint2 u;
  u.x = mm::pack2(acc.x * inv, acc.y * inv);
  u.y = mm::pack2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.out + at * D + c) = u;
}

// How a call is cut: rows per CTA, and positions per chunk.
struct AttnPlan {
  int wm, row_tiles, chunk, chunks;
};

static AttnPlan attn_plan(int n_seqs, int HQ, int HKV, int D, int max_nodes, int max_len) {
  AttnPlan p;
  const int rows = max_nodes * (HQ / HKV);
  p.wm = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  p.row_tiles = (rows + 16 * p.wm - 1) / (16 * p.wm);
  const int64_t units = (int64_t)n_seqs * HKV * p.row_tiles;
  const int64_t want = 148 * 24;                      // CTAs, for an even finish
  int64_t chunk = (units * max_len + want - 1) / want;
  chunk = (chunk + 63) / 64 * 64;
  if (chunk < 256) chunk = 256;
  if (chunk > 4096) chunk = 4096;
  p.chunk = (int)chunk;
  p.chunks = (max_len + p.chunk - 1) / p.chunk;
  if (p.chunks < 1) p.chunks = 1;
  return p;
}

static int64_t attn_workspace(const AttnPlan& p, int64_t n_tokens, int HQ, int D) {
  return p.chunks == 1 ? 0 : p.chunks * n_tokens * HQ * (4ll * D + 8);
}

template <int D, int WM, int WN, int BN>
static int launch_attention(const AttnArgs& a, cudaStream_t s) {
  const int pages = a.chunk / a.block_size + 2;
  const size_t bytes = sizeof(AttnSmem<D, WM, WN, BN>) + pages * sizeof(int);
  auto fn = attention_tree_kernel<D, WM, WN, BN>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
      cudaSuccess)
    return check_launch("gdn_attention_tree");
  const dim3 grid((unsigned)(a.n_seqs * a.HKV * a.row_tiles), (unsigned)a.chunks);
  fn<<<grid, 32 * WM * WN, bytes, s>>>(a);
  if (a.chunks > 1) {
    const int items = a.max_nodes * a.HQ * (D / 4);
    attention_join_kernel<D><<<dim3((items + 255) / 256, a.n_seqs), 256, 0, s>>>(a);
  }
  return check_launch("gdn_attention_tree");
}

}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_attention_tree_workspace_bytes(int64_t n_tokens, int32_t n_seqs,
                                                      int32_t num_q_heads, int32_t num_kv_heads,
                                                      int32_t head_dim, int32_t max_nodes,
                                                      int32_t max_len) {
  if (n_tokens <= 0 || n_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      max_nodes <= 0 || max_len <= 0)
    return 0;
  return attn_workspace(attn_plan(n_seqs, num_q_heads, num_kv_heads, head_dim, max_nodes, max_len),
                        n_tokens, num_q_heads, head_dim);
}

extern "C" int gdn_attention_tree(const void* q, int64_t q_row_stride, const void* k_cache,
                                  const void* v_cache, int64_t block_stride, int64_t token_stride,
                                  int64_t head_stride, int64_t num_blocks, int32_t block_size,
                                  const int32_t* block_tables, int64_t table_stride,
                                  int32_t max_blocks, const int32_t* context_lens,
                                  const int32_t* cu_seqlens, int32_t n_seqs,
                                  const int32_t* parents, int32_t max_nodes, int64_t n_tokens,
                                  int32_t max_len, void* out, int32_t num_q_heads,
                                  int32_t num_kv_heads, int32_t head_dim, float scale,
                                  void* workspace, int64_t workspace_bytes, int32_t* status,
                                  void* stream) {
  clear_error();
  const char* fn = "gdn_attention_tree";
  GDN_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && num_q_heads > 0 && num_kv_heads > 0 &&
                  max_nodes >= 0 && max_len >= 0,
              "%s: bad sizes (n_seqs=%d, n_tokens=%lld, HQ=%d, HKV=%d)", fn, n_seqs,
              (long long)n_tokens, num_q_heads, num_kv_heads);
  GDN_REQUIRE(num_q_heads % num_kv_heads == 0, "%s: %d query heads are not a multiple of %d kv heads",
              fn, num_q_heads, num_kv_heads);
  GDN_UNSUPPORTED(head_dim == 64 || head_dim == 128 || head_dim == 256,
                  "%s: head dim %d unsupported (64, 128, 256)", fn, head_dim);
  GDN_UNSUPPORTED(max_nodes <= kMaxTreeNodes, "%s: %d nodes in a tree (max %d)", fn, max_nodes,
                  kMaxTreeNodes);
  GDN_REQUIRE(num_blocks >= 0 && block_size > 0 && max_blocks >= 0 && table_stride >= max_blocks,
              "%s: bad cache or block table sizes", fn);
  GDN_REQUIRE(q_row_stride >= (int64_t)num_q_heads * head_dim,
              "%s: row stride smaller than the heads it holds", fn);
  GDN_REQUIRE(head_stride >= head_dim && token_stride >= head_dim && block_stride >= head_dim,
              "%s: cache strides smaller than a head", fn);
  if (n_seqs == 0 || n_tokens == 0 || max_nodes == 0) return GDN_OK;
  GDN_REQUIRE(max_len >= 1, "%s: max_len %d leaves no room for a node", fn, max_len);
  GDN_REQUIRE(q && k_cache && v_cache && block_tables && context_lens && cu_seqlens && parents && out,
              "%s: null pointer", fn);
  GDN_UNSUPPORTED(((q_row_stride | block_stride | token_stride | head_stride) & 7) == 0 &&
                      aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out),
                  "%s: operands and strides must be 16-byte aligned", fn);
  GDN_UNSUPPORTED(max_len <= (1 << 30), "%s: max_len %d too large", fn, max_len);
  const AttnPlan p = attn_plan(n_seqs, num_q_heads, num_kv_heads, head_dim, max_nodes, max_len);
  const int64_t need = attn_workspace(p, n_tokens, num_q_heads, head_dim);
  GDN_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && aligned16(workspace)),
              "%s: workspace of %lld bytes needed (16-byte aligned), got %lld", fn, (long long)need,
              (long long)workspace_bytes);
  GDN_UNSUPPORTED((int64_t)n_seqs * num_kv_heads * p.row_tiles < (1ll << 31) && p.chunks <= 65535 &&
                      n_seqs <= 65535,
                  "%s: too many sequences, heads or chunks", fn);
  AttnArgs a{(const bf16*)q, q_row_stride, (const bf16*)k_cache, (const bf16*)v_cache,
             block_stride, token_stride, head_stride, num_blocks, block_size, block_tables,
             table_stride, max_blocks, context_lens, cu_seqlens, n_seqs, parents, max_nodes,
             n_tokens, max_len, (bf16*)out, num_q_heads, num_kv_heads,
             scale * 1.4426950408889634f, p.chunk, p.chunks, p.row_tiles, (float*)workspace,
             nullptr, status};
  a.part_ml = reinterpret_cast<float2*>(a.part_o + p.chunks * n_tokens * num_q_heads * head_dim);
  cudaStream_t s = (cudaStream_t)stream;
#define GDN_AT(D, BN)                                                   \
  if (p.wm == 1) return launch_attention<D, 1, 4, BN < 64 ? 64 : BN>(a, s); \
  if (p.wm == 2) return launch_attention<D, 2, 2, BN>(a, s);            \
  return launch_attention<D, 4, 1, BN>(a, s)
  if (head_dim == 64) { GDN_AT(64, 64); }
  if (head_dim == 128) { GDN_AT(128, 64); }
  GDN_AT(256, 32);
#undef GDN_AT
}
