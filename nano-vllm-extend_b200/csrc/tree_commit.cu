// Taking an accepted path over: the conv window and the recurrent state of each
// sequence's slot, as if the path's tokens had been decoded one by one.
//
// accepted[r] is the last accepted node of sequence r (its ancestors stand with
// it), -1 where none was.  For the path's nodes in order, per v-head, as in
// recurrent.cu:
//   S <- S e^g;  d = beta (v - S^T k^);  S <- S + k^ (x) d
// and the window keeps the last K-1 of (window, the path's projection rows).
//
// HBM-bound for short paths: the state in and out once, 128 KiB per (sequence,
// v-head) at head dim 128.  Each token costs 3 fp32 operations per element of
// the state, so the arithmetic catches up at about ten accepted tokens.
//
// A CTA owns one (sequence, v-head); a warp owns 16 value columns and keeps its
// part of the state in registers from the one read to the one write: a lane
// holds 4 columns (float4) of DK / 8 rows.  S^T k^ then needs a sum over the 8
// lanes of a column group only, by shuffles: no CTA barrier between tokens.
// Keys and values are staged for eight tokens at a time.  The conv windows are
// rolled by further CTAs of the same launch.
#include "tree.cuh"

namespace gdn {

constexpr int kCommitTokens = 8;

struct CommitConv {
  const bf16* x;
  int64_t xs;
  bf16* pool;
  int64_t slot_stride;
  int channels, kernel, ctas;   // ctas: CTAs per sequence
};

template <int DK, int DV>
__global__ void __launch_bounds__(DV * 2) commit_tree_kernel(
    const bf16* __restrict__ k, int64_t ks, const bf16* __restrict__ v, int64_t vs,
    const float* __restrict__ g, const bf16* __restrict__ beta, float* __restrict__ pool,
    int64_t slot_stride, int64_t num_slots, const int64_t* __restrict__ ids,
    const int32_t* __restrict__ cu, const int32_t* __restrict__ parents,
    const int32_t* __restrict__ accepted, int max_nodes, int64_t n_tokens, int n_seqs, int HK,
    int HV, const CommitConv conv, int32_t* status) {
  constexpr int NT = DV * 2, NW = NT / 32, RPL = DK / 8, KP = RPL + 4;
  __shared__ __align__(16) float sk[kCommitTokens][8 * KP];   // row group rl at rl * KP
  __shared__ __align__(16) float sv[kCommitTokens][DV];
  __shared__ float seg[kCommitTokens], sbeta[kCommitTokens];
  __shared__ int spar[kMaxTreeNodes], spath[kMaxTreeNodes], sdepth;

  const int64_t units = (int64_t)n_seqs * HV;
  const bool is_conv = blockIdx.x >= units;
  const int seq = is_conv ? (int)((blockIdx.x - units) / conv.ctas) : (int)(blockIdx.x / HV);
  const int tid = threadIdx.x;
  int64_t start;
  int n;
  const int64_t slot = ids[seq];
  if (!tree_rows(cu, seq, n_tokens, max_nodes, status, start, n)) return;
  const int last = accepted[seq];
  if (last < -1 || last >= n) {
    if (status) atomicOr(status, GDN_STATUS_BAD_TREE);
    return;
  }
  if (last < 0) return;
  if (!slot_ok(slot, num_slots, status)) return;
  // a malformed tree leaves both pools alone (every CTA of the sequence sees all of it)
  bool malformed = false;
  if (tid < n) {
    const int p = parents[start + tid];
    malformed = p < -1 || p >= tid;
    spar[tid] = p;
  }
  if (__syncthreads_or(malformed)) {
    if (status && tid == 0) atomicOr(status, GDN_STATUS_BAD_TREE);
    return;
  }

  if (is_conv) {
    const int c = (int)((blockIdx.x - units) % conv.ctas) * NT + tid;
    if (c >= conv.channels) return;
    const int T = conv.kernel - 1;
    bf16* sp = conv.pool + slot * conv.slot_stride + (int64_t)c * T;
    bf16 nw[3];
    int at = last, m = 0;              // the path's newest T rows, newest first
    for (; m < T && at >= 0; ++m) {
      nw[m] = conv.x[(start + at) * conv.xs + c];
      at = spar[at];
    }
    bf16 old[3];
    for (int j = 0; j + m < T; ++j) old[j] = sp[j + m];
    for (int j = 0; j < T; ++j) sp[j] = j + m < T ? old[j] : nw[T - 1 - j];
    return;
  }

  const int h = (int)(blockIdx.x - (int64_t)seq * HV), hk = h / (HV / HK);
  const int warp = tid >> 5, lane = tid & 31, cl = lane & 3, rl = lane >> 2;
  const int c = warp * 16 + 4 * cl;
  float* sp = pool + slot * slot_stride + (int64_t)h * DK * DV + (int64_t)(rl * RPL) * DV + c;
  float4 s[RPL];
#pragma unroll
  for (int i = 0; i < RPL; ++i) s[i] = __ldcs(reinterpret_cast<const float4*>(sp + i * DV));

  if (tid == 0) {
    int m = 0;
    for (int at = last; at >= 0; at = spar[at]) ++m;
    sdepth = m;
    for (int at = last; at >= 0; at = spar[at]) spath[--m] = at;
  }
  __syncthreads();
  const int depth = sdepth;

  for (int t0 = 0; t0 < depth; t0 += kCommitTokens) {
    const int m = min(kCommitTokens, depth - t0);
    for (int i = warp; i < m; i += NW) {      // a warp per token
      const int64_t row = start + spath[t0 + i];
      float x[DK / 32], ss = 0.f;
#pragma unroll
      for (int e = 0; e < DK / 32; ++e) {
        x[e] = bf2f(k[row * ks + (int64_t)hk * DK + lane + 32 * e]);
        ss = fmaf(x[e], x[e], ss);
      }
      const float nk = rsqrtf(warp_sum(ss) + 1e-6f);
#pragma unroll
      for (int e = 0; e < DK / 32; ++e) {
        const int r = lane + 32 * e;
        sk[i][(r / RPL) * KP + r % RPL] = x[e] * nk;
      }
#pragma unroll
      for (int e = 0; e < DV / 32; ++e)
        sv[i][lane + 32 * e] = bf2f(v[row * vs + (int64_t)h * DV + lane + 32 * e]);
      if (lane == 0) {
        seg[i] = expf(g[row * HV + h]);
        sbeta[i] = bf2f(beta[row * HV + h]);
      }
    }
    __syncthreads();
    for (int i = 0; i < m; ++i) {
      const float* kr = &sk[i][rl * KP];
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < RPL; r += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(kr + r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ke = e == 0 ? kk.x : e == 1 ? kk.y : e == 2 ? kk.z : kk.w;
          a.x = fmaf(s[r + e].x, ke, a.x);
          a.y = fmaf(s[r + e].y, ke, a.y);
          a.z = fmaf(s[r + e].z, ke, a.z);
          a.w = fmaf(s[r + e].w, ke, a.w);
        }
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        a.x += __shfl_xor_sync(0xffffffffu, a.x, o);
        a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
        a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
        a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
      }
      const float eg = seg[i], bt = sbeta[i];
      const float4 vv = *reinterpret_cast<const float4*>(&sv[i][c]);
      const float4 d = make_float4(bt * (vv.x - eg * a.x), bt * (vv.y - eg * a.y),
                                   bt * (vv.z - eg * a.z), bt * (vv.w - eg * a.w));
#pragma unroll
      for (int r = 0; r < RPL; r += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(kr + r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ke = e == 0 ? kk.x : e == 1 ? kk.y : e == 2 ? kk.z : kk.w;
          s[r + e].x = fmaf(ke, d.x, s[r + e].x * eg);
          s[r + e].y = fmaf(ke, d.y, s[r + e].y * eg);
          s[r + e].z = fmaf(ke, d.z, s[r + e].z * eg);
          s[r + e].w = fmaf(ke, d.w, s[r + e].w * eg);
        }
      }
    }
    if (t0 + kCommitTokens < depth) __syncthreads();   // the staging buffers are free
  }
#pragma unroll
  for (int i = 0; i < RPL; ++i) __stcs(reinterpret_cast<float4*>(sp + i * DV), s[i]);
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_commit_tree(const void* x, int64_t x_row_stride, const void* k,
                               int64_t k_row_stride, const void* v, int64_t v_row_stride,
                               const float* g, const void* beta, void* conv_pool,
                               int64_t conv_slot_stride, int32_t channels, int32_t kernel,
                               float* s_pool, int64_t slot_stride, int64_t num_slots,
                               const int64_t* ids, const int32_t* cu_seqlens, int32_t n_seqs,
                               const int32_t* parents, const int32_t* accepted, int32_t max_nodes,
                               int64_t n_tokens, int32_t num_k_heads, int32_t num_v_heads,
                               int32_t head_k_dim, int32_t head_v_dim, int32_t* status,
                               void* stream) {
  clear_error();
  const char* fn = "gdn_commit_tree";
  GDN_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && num_k_heads > 0 && num_v_heads > 0 &&
                  max_nodes >= 0 && channels > 0,
              "%s: bad sizes (n_seqs=%d, n_tokens=%lld, HK=%d, HV=%d, channels=%d)", fn, n_seqs,
              (long long)n_tokens, num_k_heads, num_v_heads, channels);
  GDN_REQUIRE(num_v_heads % num_k_heads == 0, "%s: num_v_heads %d not a multiple of num_k_heads %d",
              fn, num_v_heads, num_k_heads);
  GDN_UNSUPPORTED(head_k_dim == head_v_dim && (head_v_dim == 64 || head_v_dim == 128),
                  "%s: head dims (%d, %d) unsupported", fn, head_k_dim, head_v_dim);
  GDN_UNSUPPORTED(kernel >= 2 && kernel <= 4, "%s: kernel %d unsupported (2..4)", fn, kernel);
  GDN_UNSUPPORTED(max_nodes <= kMaxTreeNodes, "%s: %d nodes in a tree (max %d)", fn, max_nodes,
                  kMaxTreeNodes);
  GDN_REQUIRE(x_row_stride >= channels && k_row_stride >= (int64_t)num_k_heads * head_k_dim &&
                  v_row_stride >= (int64_t)num_v_heads * head_v_dim,
              "%s: row stride smaller than the row it holds", fn);
  GDN_REQUIRE(num_slots > 0 && slot_stride >= (int64_t)num_v_heads * head_k_dim * head_v_dim &&
                  slot_stride % 4 == 0,
              "%s: slot_stride %lld must be >= HV*DK*DV and a multiple of 4", fn,
              (long long)slot_stride);
  GDN_REQUIRE(conv_slot_stride >= (int64_t)channels * (kernel - 1), "%s: conv_slot_stride too small",
              fn);
  if (n_seqs == 0 || n_tokens == 0 || max_nodes == 0) return GDN_OK;
  GDN_REQUIRE(x && k && v && g && beta && conv_pool && s_pool && ids && cu_seqlens && parents &&
                  accepted,
              "%s: null pointer", fn);
  GDN_REQUIRE(aligned16(s_pool), "%s: s_pool must be 16-byte aligned", fn);
  const int nt = head_v_dim * 2;
  const CommitConv conv{(const bf16*)x, x_row_stride, (bf16*)conv_pool, conv_slot_stride, channels,
                        kernel, (channels + nt - 1) / nt};
  const int64_t ctas = (int64_t)n_seqs * (num_v_heads + conv.ctas);
  GDN_UNSUPPORTED(ctas < (1ll << 31), "%s: too many (sequence, head) units", fn);
  cudaStream_t s = (cudaStream_t)stream;
#define GDN_CM(D)                                                                                \
  commit_tree_kernel<D, D><<<(unsigned)ctas, 2 * D, 0, s>>>(                                     \
      (const bf16*)k, k_row_stride, (const bf16*)v, v_row_stride, g, (const bf16*)beta, s_pool,  \
      slot_stride, num_slots, ids, cu_seqlens, parents, accepted, max_nodes, n_tokens, n_seqs,   \
      num_k_heads, num_v_heads, conv, status)
  if (head_v_dim == 128) GDN_CM(128);
  else GDN_CM(64);
#undef GDN_CM
  return check_launch(fn);
}
