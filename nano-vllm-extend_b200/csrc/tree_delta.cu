// The gated delta rule along trees of drafted tokens: every node's output from
// its sequence's stored state, which is read once and left as it is.
//
// The recurrence (as in recurrent.cu) along a node's ancestors, S_0 the stored
// state, p(i) the parent of node i:
//   S'_i = e^{g_i} S_p(i);  d_i = beta_i (v_i - S'_i^T k_i);  S_i = S'_i + k_i (x) d_i
//   o_i = S_i^T q_i                    (q, k l2-normed, q scaled)
// A tree branches, so no single running state serves it.  Unrolled over the
// ancestors j of i, with D_ij the product of e^{g} on the path (j, i] and D_i0
// that from the root:
//   d_i = beta_i (v_i - D_i0 S_0^T k_i) - sum_{j < i, ancestor} A_ij d_j,  A_ij = beta_i D_ij k_i.k_j
//   o_i = D_i0 S_0^T q_i + sum_{j <= i, ancestor} M_ij d_j,                M_ij = D_ij q_i.k_j
// S_0 enters through X = [K; Q] S_0 alone: a product whose columns (the state's
// value columns) are independent, as is everything after it.
//
// HBM: the state is the traffic, 64 KiB per (sequence, v-head) at head dim 128,
// read once; q, k, v, z and the output are 2 bytes x n nodes x 128 each.
//
// One CTA per (sequence, v-head), a warp per 16 value columns.  Products are
// computed transposed, X^T = S_0^T [K; Q]^T with mma.sync m16n8k16: 16 value
// columns by 8 nodes, so few nodes waste little, and S_0^T's fragments load
// straight from global memory into registers (float2 along a row: rows g and
// g + 8 of the fragment are the value columns 2g and 2g + 1), all 64 KiB of the
// CTA in flight before anything else is done.  The results' layout is that of
// the next product's A operand (node index = its k), so X, d and o never leave
// the warp's registers.  fp32 factors enter the bf16 products as hi + lo pairs
// (S_0: 2 products with the exact bf16 q / k; A, M with d: 3), 16 mantissa bits
// each under fp32 sums, well inside the output's bf16 step; the norms, decays,
// gram factors and the substitution over a block's 16 nodes are fp32.
//
// A node whose own d is not finite (a NaN or infinity in its row) must not reach
// nodes that do not descend from it: zero coefficients would still turn it into
// NaN, so its d is set to zero for the products and its own and its descendants'
// outputs are set to NaN at the end.
#include "mma_util.cuh"
#include "tc_util.cuh"
#include "tree.cuh"

namespace gdn {

template <int DK, int DV, int TN>
struct TreeDeltaSmem {
  static constexpr int KP = DK + 8;                  // q / k row pitch: conflict-free ldmatrix
  static constexpr int TB = TN < 16 ? TN : 16;       // substitution block
  static constexpr int AW = TN < 16 ? 16 : TN;       // factor row width (k extent of an MMA)
  static constexpr int AP = AW + 8;
  static constexpr int NW = DV / 16;
  bf16 kq[2 * TN][KP];                               // raw rows: keys, then queries
  bf16 ahi[TN][AP], alo[TN][AP];                     // -A
  bf16 mhi[TN][AP], mlo[TN][AP];                     // M
  float at[TN / TB][TB][TB];                         // -A's diagonal blocks, at[.][i][j] = -A_ji
  float dec[TN][TN + 1];                             // D_ij, zero where j is no ancestor of i
  float d0[TN], eg[TN], beta[TN];
  float norm[2 * TN];                                // 1 / |k|, scale / |q|
  float ssum[NW][TN];
  int par[TN];
};

// Element d0..d0+7 of a head row; rows may be unaligned (vec false).
__device__ __forceinline__ uint4 load8(const bf16* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint4 u;
  bf16* h = reinterpret_cast<bf16*>(&u);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = p[e];
  return u;
}

template <int DK, int DV, int TN, bool NORM>
__global__ void __launch_bounds__(DV * 2) tree_delta_kernel(
    const bf16* __restrict__ q, int64_t qs, const bf16* __restrict__ k, int64_t ks,
    const bf16* __restrict__ v, int64_t vs, const float* __restrict__ g,
    const bf16* __restrict__ beta, const float* __restrict__ pool, int64_t slot_stride,
    int64_t num_slots, const int64_t* __restrict__ ids, const int32_t* __restrict__ cu,
    const int32_t* __restrict__ parents, int max_nodes, int64_t n_tokens, bf16* __restrict__ out,
    int HK, int HV, float scale, const bf16* __restrict__ z, int64_t zs,
    const bf16* __restrict__ nw, float eps, bool vec, int32_t* status) {
  using S = TreeDeltaSmem<DK, DV, TN>;
  constexpr int NT = DV * 2, NW = S::NW, KB = DK / 16, KT = TN / 8, TB = S::TB, BT = TB / 8;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);

  const int seq = blockIdx.x / HV, h = blockIdx.x - seq * HV;
  const int hk = h / (HV / HK);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  int64_t start;
  int n;
  const int64_t slot = ids[seq];
  if (!tree_rows(cu, seq, n_tokens, max_nodes, status, start, n) || n == 0) return;
  if (!slot_ok(slot, num_slots, status)) return;

  // the whole state into registers: value columns c, c + 1; rows 16 kb + 2t, +1, +8, +9
  const int c = warp * 16 + 2 * gr;
  const float* sp = pool + slot * slot_stride + (int64_t)h * DK * DV + (2 * tq) * DV + c;
  float2 st[KB][4];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    st[kb][0] = __ldcs(reinterpret_cast<const float2*>(sp + (kb * 16) * DV));
    st[kb][1] = __ldcs(reinterpret_cast<const float2*>(sp + (kb * 16 + 1) * DV));
    st[kb][2] = __ldcs(reinterpret_cast<const float2*>(sp + (kb * 16 + 8) * DV));
    st[kb][3] = __ldcs(reinterpret_cast<const float2*>(sp + (kb * 16 + 9) * DV));
  }

  // q / k rows (zero rows behind the last node), factors' zero columns, scalars
  for (int i = tid; i < 2 * TN * (DK / 8); i += NT) {
    const int row = i / (DK / 8), ch = (i - row * (DK / 8)) * 8;
    const int node = row % TN;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (node < n)
      u = row < TN ? load8(k + (start + node) * ks + (int64_t)hk * DK + ch, vec)
                   : load8(q + (start + node) * qs + (int64_t)hk * DK + ch, vec);
    *reinterpret_cast<uint4*>(&sm.kq[row][ch]) = u;
  }
  if constexpr (TN < 16) {
    for (int i = tid; i < TN * 8; i += NT) {
      const bf16 zero = f2bf(0.f);
      sm.ahi[i / 8][8 + i % 8] = sm.alo[i / 8][8 + i % 8] = zero;
      sm.mhi[i / 8][8 + i % 8] = sm.mlo[i / 8][8 + i % 8] = zero;
    }
  }
  if (tid < TN) {
    const bool on = tid < n;
    sm.par[tid] = on ? tree_parent(parents[start + tid], tid, status) : -1;
    sm.eg[tid] = on ? expf(g[(start + tid) * HV + h]) : 0.f;
    sm.beta[tid] = on ? bf2f(beta[(start + tid) * HV + h]) : 0.f;
  }
  // this thread's values: nodes 8 t8 + 2t, +1, columns c, c + 1
  uint32_t vr[KT][2];
#pragma unroll
  for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int node = t8 * 8 + 2 * tq + e;
      vr[t8][e] = node < n ? *reinterpret_cast<const uint32_t*>(v + (start + node) * vs +
                                                                (int64_t)h * DV + c)
                           : 0u;
    }
  __syncthreads();

  // decays: thread j owns column j (d from node j down), thread TN the root's
  if (tid <= TN) {
    float prev = 0.f;
    for (int i = 0; i < n; ++i) {
      const int p = sm.par[i];
      float d;
      if (tid == TN) {
        d = sm.eg[i] * (p < 0 ? 1.f : p == i - 1 ? prev : sm.d0[p]);
        sm.d0[i] = d;
      } else {
        const float up = p < 0 ? 0.f : p == i - 1 ? prev : sm.dec[p][tid];
        d = i == tid ? 1.f : up == 0.f ? 0.f : sm.eg[i] * up;
        sm.dec[i][tid] = d;
      }
      prev = d;
    }
    for (int i = n; i < TN; ++i) {
      if (tid == TN) sm.d0[i] = 0.f;
      else sm.dec[i][tid] = 0.f;
    }
  }
  // norms, a warp per row
  for (int row = warp; row < 2 * TN; row += NW) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < DK / 32; ++e) {
      const float x = bf2f(sm.kq[row][lane + 32 * e]);
      ss = fmaf(x, x, ss);
    }
    ss = warp_sum(ss);
    if (lane == 0) sm.norm[row] = rsqrtf(ss + 1e-6f) * (row < TN ? 1.f : scale);
  }
  __syncthreads();

  // gram tiles [K; Q] K^T -> the factors -A and M
  const uint32_t kq0 = tc::smem_u32(&sm.kq[0][0]);
  for (int tile = warp; tile < (2 * TN / 16) * KT; tile += NW) {
    const int mt = tile / KT, nt = tile - mt * KT;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t a_addr = kq0 + ((mt * 16 + (lane & 15)) * S::KP + (lane >> 4) * 8) * 2;
    const uint32_t b_addr = kq0 + ((nt * 8 + (lane & 7)) * S::KP + (lane >> 3) * 8) * 2;
#pragma unroll
    for (int kb = 0; kb < KB; kb += 2) {
      uint32_t a[4], b[4];
      mm::ldsm4(b, b_addr + kb * 32);
      mm::ldsm4(a, a_addr + kb * 32);
      mm::mma16816(acc, a, b[0], b[1]);
      mm::ldsm4(a, a_addr + kb * 32 + 32);
      mm::mma16816(acc, a, b[2], b[3]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = mt * 16 + gr + (e >> 1) * 8, i = nt * 8 + 2 * tq + (e & 1);
      const int j = row % TN;
      const float d = sm.dec[j][i];
      float f = d == 0.f ? 0.f : d * sm.norm[i] * sm.norm[row] * acc[e];
      if (row < TN) {
        f = i < j ? -sm.beta[j] * f : 0.f;
        if (i / TB == j / TB) sm.at[i / TB][i % TB][j % TB] = f;
        const bf16 hi = f2bf(f);
        sm.ahi[j][i] = hi;
        sm.alo[j][i] = f2bf(f - bf2f(hi));
      } else {
        const bf16 hi = f2bf(f);
        sm.mhi[j][i] = hi;
        sm.mlo[j][i] = f2bf(f - bf2f(hi));
      }
    }
  }

  // X^T = S_0^T [K; Q]^T
  float acc[2 * KT][4];
#pragma unroll
  for (int t8 = 0; t8 < 2 * KT; ++t8)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t8][e] = 0.f;
  const uint32_t x_addr = kq0 + (((lane >> 4) * 8 + (lane & 7)) * S::KP + ((lane >> 3) & 1) * 8) * 2;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    uint32_t hi[4], lo[4];
    mm::split2(st[kb][0].x, st[kb][1].x, hi[0], lo[0]);
    mm::split2(st[kb][0].y, st[kb][1].y, hi[1], lo[1]);
    mm::split2(st[kb][2].x, st[kb][3].x, hi[2], lo[2]);
    mm::split2(st[kb][2].y, st[kb][3].y, hi[3], lo[3]);
#pragma unroll
    for (int t8 = 0; t8 < 2 * KT; t8 += 2) {
      uint32_t b[4];
      mm::ldsm4(b, x_addr + (t8 * 8 * S::KP + kb * 16) * 2);
      mm::mma16816(acc[t8], hi, b[0], b[1]);
      mm::mma16816(acc[t8], lo, b[0], b[1]);
      mm::mma16816(acc[t8 + 1], hi, b[2], b[3]);
      mm::mma16816(acc[t8 + 1], lo, b[2], b[3]);
    }
  }
  // right sides (keys) and the state's part of the outputs (queries)
#pragma unroll
  for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int node = t8 * 8 + 2 * tq + e;
      const float b = sm.beta[node], f = sm.d0[node];
      const float fk = f * sm.norm[node], fq = f * sm.norm[TN + node];
      const float v0 = __uint_as_float(vr[t8][e] << 16), v1 = __uint_as_float(vr[t8][e] & 0xffff0000u);
      acc[t8][e] = node < n ? b * (v0 - fk * acc[t8][e]) : 0.f;
      acc[t8][2 + e] = node < n ? b * (v1 - fk * acc[t8][2 + e]) : 0.f;
      acc[KT + t8][e] *= fq;
      acc[KT + t8][2 + e] *= fq;
    }
  __syncthreads();                                   // the factors are complete

  unsigned long long bad = 0;
#pragma unroll
  for (int blk = 0; blk < TN / TB; ++blk) {
    if (blk * TB < n) {
      // substitution within the block: node i's d to the quad, then into later nodes
#pragma unroll
      for (int i = 0; i < TB; ++i) {
        if (blk * TB + i < n) {
          const int t8 = blk * BT + i / 8, e = i & 1, from = (lane & ~3) | ((i & 7) >> 1);
          float d0v = __shfl_sync(0xffffffffu, acc[t8][e], from);
          float d1v = __shfl_sync(0xffffffffu, acc[t8][2 + e], from);
          if (!(fabsf(d0v) <= 3.0e38f && fabsf(d1v) <= 3.0e38f)) {
            bad |= 1ull << (blk * TB + i);
            d0v = d1v = 0.f;
            if (lane == from) acc[t8][e] = acc[t8][2 + e] = 0.f;
          }
#pragma unroll
          for (int u = i / 8; u < BT; ++u) {
            const float2 a = *reinterpret_cast<const float2*>(&sm.at[blk][i][u * 8 + 2 * tq]);
            float(&r)[4] = acc[blk * BT + u];
            r[0] = fmaf(a.x, d0v, r[0]);
            r[1] = fmaf(a.y, d0v, r[1]);
            r[2] = fmaf(a.x, d1v, r[2]);
            r[3] = fmaf(a.y, d1v, r[3]);
          }
        }
      }
      // this block's d as an A operand, into the later blocks and the outputs
      uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < BT; ++u) {
        mm::split2(acc[blk * BT + u][0], acc[blk * BT + u][1], hi[2 * u], lo[2 * u]);
        mm::split2(acc[blk * BT + u][2], acc[blk * BT + u][3], hi[2 * u + 1], lo[2 * u + 1]);
      }
      // lanes 0-15 give the hi factor's rows, 16-31 the lo factor's
      const int frow = lane & 7, fcol = blk * TB + ((lane >> 3) & 1) * 8;
#pragma unroll
      for (int t8 = (blk + 1) * BT; t8 < KT; ++t8) {
        uint32_t b[4];
        mm::ldsm4(b, tc::smem_u32(lane < 16 ? &sm.ahi[t8 * 8 + frow][fcol]
                                            : &sm.alo[t8 * 8 + frow][fcol]));
        mm::mma16816(acc[t8], hi, b[0], b[1]);
        mm::mma16816(acc[t8], lo, b[0], b[1]);
        mm::mma16816(acc[t8], hi, b[2], b[3]);
      }
#pragma unroll
      for (int t8 = blk * BT; t8 < KT; ++t8) {
        uint32_t b[4];
        mm::ldsm4(b, tc::smem_u32(lane < 16 ? &sm.mhi[t8 * 8 + frow][fcol]
                                            : &sm.mlo[t8 * 8 + frow][fcol]));
        mm::mma16816(acc[KT + t8], hi, b[0], b[1]);
        mm::mma16816(acc[KT + t8], lo, b[0], b[1]);
        mm::mma16816(acc[KT + t8], hi, b[2], b[3]);
      }
    }
  }
  bad = (unsigned long long)__reduce_or_sync(0xffffffffu, (unsigned)(bad >> 32)) << 32 |
        __reduce_or_sync(0xffffffffu, (unsigned)bad);
  if (bad) {
#pragma unroll
    for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        for (int j = t8 * 8 + 2 * tq + e; j >= 0; j = sm.par[j])
          if (bad >> j & 1) {
            acc[KT + t8][e] = acc[KT + t8][2 + e] = __int_as_float(0x7fffffff);
            break;
          }
  }

  if constexpr (NORM) {
#pragma unroll
    for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float ss = acc[KT + t8][e] * acc[KT + t8][e] + acc[KT + t8][2 + e] * acc[KT + t8][2 + e];
        ss += __shfl_xor_sync(0xffffffffu, ss, 4);
        ss += __shfl_xor_sync(0xffffffffu, ss, 8);
        ss += __shfl_xor_sync(0xffffffffu, ss, 16);
        if (gr == 0) sm.ssum[warp][t8 * 8 + 2 * tq + e] = ss;
      }
    __syncthreads();
  }
  float w0 = 1.f, w1 = 1.f;
  if constexpr (NORM) {
    w0 = bf2f(nw[c]);
    w1 = bf2f(nw[c + 1]);
  }
#pragma unroll
  for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int node = t8 * 8 + 2 * tq + e;
      if (node >= n) continue;
      float o0 = acc[KT + t8][e], o1 = acc[KT + t8][2 + e];
      if constexpr (NORM) {
        float tot = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) tot += sm.ssum[i][node];
        const float inv = rsqrtf(tot * (1.f / DV) + eps);
        const uint32_t zr = *reinterpret_cast<const uint32_t*>(z + (start + node) * zs +
                                                               (int64_t)h * DV + c);
        const float z0 = __uint_as_float(zr << 16), z1 = __uint_as_float(zr & 0xffff0000u);
        o0 = o0 * inv * w0 * conv_silu(z0);
        o1 = o1 * inv * w1 * conv_silu(z1);
      }
      *reinterpret_cast<uint32_t*>(out + ((start + node) * HV + h) * DV + c) = mm::pack2(o0, o1);
    }
}

template <int D, int TN>
static int launch_tree_delta(unsigned units, cudaStream_t s, const bf16* q, int64_t qs,
                             const bf16* k, int64_t ks, const bf16* v, int64_t vs, const float* g,
                             const bf16* beta, const float* pool, int64_t slot_stride,
                             int64_t num_slots, const int64_t* ids, const int32_t* cu,
                             const int32_t* parents, int max_nodes, int64_t n_tokens, bf16* out,
                             int HK, int HV, float scale, const bf16* z, int64_t zs,
                             const bf16* nw, float eps, bool vec, int32_t* status) {
  constexpr size_t bytes = sizeof(TreeDeltaSmem<D, D, TN>);
  auto fn = z != nullptr ? tree_delta_kernel<D, D, TN, true> : tree_delta_kernel<D, D, TN, false>;
  if (bytes > 48 * 1024 &&
      cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
          cudaSuccess)
    return check_launch("gdn_delta_rule_tree");
  fn<<<units, 2 * D, bytes, s>>>(q, qs, k, ks, v, vs, g, beta, pool, slot_stride, num_slots, ids,
                                 cu, parents, max_nodes, n_tokens, out, HK, HV, scale, z, zs, nw,
                                 eps, vec, status);
  return check_launch("gdn_delta_rule_tree");
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_delta_rule_tree(const void* q, int64_t q_row_stride, const void* k,
                                   int64_t k_row_stride, const void* v, int64_t v_row_stride,
                                   const float* g, const void* beta, const float* s_pool,
                                   int64_t slot_stride, int64_t num_slots, const int64_t* ids,
                                   const int32_t* cu_seqlens, int32_t n_seqs,
                                   const int32_t* parents, int32_t max_nodes, int64_t n_tokens,
                                   void* out, int32_t num_k_heads, int32_t num_v_heads,
                                   int32_t head_k_dim, int32_t head_v_dim, float scale,
                                   const void* z, int64_t z_row_stride, const void* norm_weight,
                                   float norm_eps, int32_t* status, void* stream) {
  clear_error();
  const char* fn = "gdn_delta_rule_tree";
  GDN_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && num_k_heads > 0 && num_v_heads > 0 && max_nodes >= 0,
              "%s: bad sizes (n_seqs=%d, n_tokens=%lld, HK=%d, HV=%d)", fn, n_seqs,
              (long long)n_tokens, num_k_heads, num_v_heads);
  GDN_REQUIRE(num_v_heads % num_k_heads == 0, "%s: num_v_heads %d not a multiple of num_k_heads %d",
              fn, num_v_heads, num_k_heads);
  GDN_UNSUPPORTED(head_k_dim == head_v_dim && (head_v_dim == 64 || head_v_dim == 128),
                  "%s: head dims (%d, %d) unsupported", fn, head_k_dim, head_v_dim);
  GDN_UNSUPPORTED(max_nodes <= kMaxTreeNodes, "%s: %d nodes in a tree (max %d)", fn, max_nodes,
                  kMaxTreeNodes);
  GDN_REQUIRE(q_row_stride >= (int64_t)num_k_heads * head_k_dim &&
                  k_row_stride >= (int64_t)num_k_heads * head_k_dim &&
                  v_row_stride >= (int64_t)num_v_heads * head_v_dim,
              "%s: row stride smaller than the heads it holds", fn);
  GDN_REQUIRE(num_slots > 0 && slot_stride >= (int64_t)num_v_heads * head_k_dim * head_v_dim &&
                  slot_stride % 4 == 0,
              "%s: slot_stride %lld must be >= HV*DK*DV and a multiple of 4", fn,
              (long long)slot_stride);
  GDN_REQUIRE(z == nullptr ||
                  (norm_weight != nullptr && z_row_stride >= (int64_t)num_v_heads * head_v_dim),
              "%s: fused norm needs norm_weight and z rows of HV*DV", fn);
  if (n_seqs == 0 || n_tokens == 0 || max_nodes == 0) return GDN_OK;
  GDN_REQUIRE(q && k && v && g && beta && s_pool && ids && cu_seqlens && parents && out,
              "%s: null pointer", fn);
  GDN_REQUIRE(aligned16(s_pool), "%s: s_pool must be 16-byte aligned", fn);
  GDN_UNSUPPORTED(v_row_stride % 2 == 0 && (z == nullptr || z_row_stride % 2 == 0) &&
                      ((uintptr_t)v | (uintptr_t)z | (uintptr_t)out) % 4 == 0,
                  "%s: v, z and out must be 4-byte aligned with even row strides", fn);
  const int64_t units = (int64_t)n_seqs * num_v_heads;
  GDN_UNSUPPORTED(units < (1ll << 31), "%s: too many (sequence, head) units", fn);
  const bool vec = aligned16(q) && aligned16(k) && q_row_stride % 8 == 0 && k_row_stride % 8 == 0;
#define GDN_TD(D, TN)                                                                             \
  return launch_tree_delta<D, TN>(                                                                \
      (unsigned)units, (cudaStream_t)stream, (const bf16*)q, q_row_stride, (const bf16*)k,        \
      k_row_stride, (const bf16*)v, v_row_stride, g, (const bf16*)beta, s_pool, slot_stride,      \
      num_slots, ids, cu_seqlens, parents, max_nodes, n_tokens, (bf16*)out, num_k_heads,          \
      num_v_heads, scale, (const bf16*)z, z_row_stride, (const bf16*)norm_weight, norm_eps, vec,  \
      status)
#define GDN_TDN(D)                                                                                \
  if (max_nodes <= 8) GDN_TD(D, 8);                                                               \
  if (max_nodes <= 16) GDN_TD(D, 16);                                                             \
  if (max_nodes <= 32) GDN_TD(D, 32);                                                             \
  GDN_TD(D, 64)
  if (head_v_dim == 128) { GDN_TDN(128); }
  GDN_TDN(64);
#undef GDN_TDN
#undef GDN_TD
}
