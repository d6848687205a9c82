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
// lanes of a column group only, by shuffles, and |k| likewise: no CTA barrier
// between tokens.  What is small is asked for before the state, behind which it would
// queue; in trees of up to kStaged nodes that is every node's key and value, whatever
// path is accepted, so that nothing waits for the path (268 -> 199 us for 256
// sequences x 32 heads of 3 to 8 nodes, floor 168).  Larger trees stage their path's
// rows, kStaged at a time.  The conv windows are rolled by further CTAs of the same launch.
#include "tc_util.cuh"
#include "tree.cuh"

namespace gdn {

constexpr int kStaged = 16;

struct CommitConv {
  const bf16* x;
  int64_t xs;
  bf16* pool;
  int64_t slot_stride;
  int channels, kernel, ctas;   // ctas: CTAs per sequence
  bool vec;                     // eight channels per thread (16-byte aligned)
};

// Eight channels' windows of T taps: M path rows (the newest first) enter.
template <int T, int M>
__device__ __forceinline__ void roll8(bf16* sp, const uint4 (&rows)[3]) {
  uint4 old[T], out[T];
#pragma unroll
  for (int j = 0; j < T; ++j) old[j] = reinterpret_cast<const uint4*>(sp)[j];
  const bf16* o = reinterpret_cast<const bf16*>(old);
  bf16* n = reinterpret_cast<bf16*>(out);
#pragma unroll
  for (int ch = 0; ch < 8; ++ch)
#pragma unroll
    for (int j = 0; j < T; ++j)
      n[ch * T + j] = j + M < T ? o[ch * T + j + M] : reinterpret_cast<const bf16*>(&rows[T - 1 - j])[ch];
#pragma unroll
  for (int j = 0; j < T; ++j) reinterpret_cast<uint4*>(sp)[j] = out[j];
}

template <int T>
__device__ __forceinline__ void roll8(bf16* sp, const uint4 (&rows)[3], int m) {
  if (m >= T) roll8<T, T>(sp, rows);
  else if (m == 1) roll8<T, 1>(sp, rows);
  else if constexpr (T > 2) roll8<T, 2>(sp, rows);
}

template <int DK, int DV>
__global__ void __launch_bounds__(DV * 2, DV == 128 ? 2 : 4) commit_tree_kernel(
    const bf16* __restrict__ k, int64_t ks, const bf16* __restrict__ v, int64_t vs,
    const float* __restrict__ g, const bf16* __restrict__ beta, float* __restrict__ pool,
    int64_t slot_stride, int64_t num_slots, const int64_t* __restrict__ ids,
    const int32_t* __restrict__ cu, const int32_t* __restrict__ parents,
    const int32_t* __restrict__ accepted, int max_nodes, int64_t n_tokens, int n_seqs, int HK,
    int HV, bool vec, const CommitConv conv, int32_t* status) {
  constexpr int NT = DV * 2, RPL = DK / 8, PK = DK / 8;
  __shared__ __align__(16) bf16 sk[kStaged][DK];
  __shared__ __align__(16) bf16 sv[kStaged][DV];
  __shared__ float sg[kMaxTreeNodes], sbeta[kMaxTreeNodes];
  __shared__ int spar[kMaxTreeNodes];

  const int64_t units = (int64_t)n_seqs * HV;
  const bool is_conv = blockIdx.x >= units;
  const int seq = is_conv ? (int)((blockIdx.x - units) / conv.ctas) : (int)(blockIdx.x / HV);
  const int tid = threadIdx.x;
  int64_t start;
  int n;
  const int64_t slot = ids[seq];
  const int last = accepted[seq];
  if (!tree_rows(cu, seq, n_tokens, max_nodes, status, start, n)) return;
  if (last < -1 || last >= n) {
    if (status) atomicOr(status, GDN_STATUS_BAD_TREE);
    return;
  }
  if (last < 0) return;
  if (!slot_ok(slot, num_slots, status)) return;
  const int h = is_conv ? 0 : (int)(blockIdx.x - (int64_t)seq * HV), hk = h / (HV / HK);

  int my_par = -1;
  if (tid < n) my_par = parents[start + tid];
  // m rows of keys and values into the staging buffers, all threads together
  const auto stage = [&](int m, const auto& node_of) {
    for (int i = tid; i < m * 2 * PK; i += NT) {
      const int r = i / (2 * PK), pc = i - r * 2 * PK, c8 = pc % PK * 8;
      const int64_t row = start + node_of(r);
      const bf16* src = pc < PK ? k + row * ks + (int64_t)hk * DK + c8
                                : v + row * vs + (int64_t)h * DV + c8;
      bf16* dst = pc < PK ? &sk[r][c8] : &sv[r][c8];
      if (vec) {
        tc::cp_async16(tc::smem_u32(dst), src, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[e] = src[e];
      }
    }
  };
  if (!is_conv) {
    if (n <= kStaged) stage(n, [](int r) { return r; });
    if (tid < n) {
      sg[tid] = g[(start + tid) * HV + h];
      sbeta[tid] = bf2f(beta[(start + tid) * HV + h]);
    }
  }

  const int warp = tid >> 5, lane = tid & 31, cl = lane & 3, rl = lane >> 2;
  const int c = warp * 16 + 4 * cl;
  float* sp = pool + slot * slot_stride + (int64_t)h * DK * DV + (int64_t)(rl * RPL) * DV + c;
  float4 s[RPL];
  if (!is_conv) {
#pragma unroll
    for (int i = 0; i < RPL; ++i) s[i] = __ldcs(reinterpret_cast<const float4*>(sp + i * DV));
  }

  // a malformed tree leaves both pools alone (every CTA of the sequence sees all of it)
  if (tid < n) spar[tid] = my_par;
  tc::cp_async_commit();
  tc::cp_async_wait<0>();
  if (__syncthreads_or(tid < n && (my_par < -1 || my_par >= tid))) {
    if (status && tid == 0) atomicOr(status, GDN_STATUS_BAD_TREE);
    return;
  }

  if (is_conv) {
    const int T = conv.kernel - 1;
    const int c0 = ((int)((blockIdx.x - units) % conv.ctas) * NT + tid) * (conv.vec ? 8 : 1);
    if (c0 >= conv.channels) return;
    bf16* to = conv.pool + slot * conv.slot_stride + (int64_t)c0 * T;
    int at = last, m = 0;              // the path's newest T rows, newest first
    if (conv.vec) {
      uint4 rows[3];
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < T && at >= 0) {
          rows[j] = *reinterpret_cast<const uint4*>(conv.x + (start + at) * conv.xs + c0);
          at = spar[at];
          ++m;
        }
      if (T == 3) roll8<3>(to, rows, m);
      else if (T == 2) roll8<2>(to, rows, m);
      else roll8<1>(to, rows, m);
      return;
    }
    bf16 nw[3], old[3];
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < T && at >= 0) {
        nw[j] = conv.x[(start + at) * conv.xs + c0];
        at = spar[at];
        ++m;
      }
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < T) old[j] = to[j];
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < T) {
        // tap j: old tap j + m, or the path's row T - 1 - j
        bf16 x = nw[0];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (j + m < T && i == j + m) x = old[i];
          if (j + m >= T && i == T - 1 - j) x = nw[i];
        }
        to[j] = x;
      }
    return;
  }

  // the path as bits: parents come before their children, so its order is theirs
  unsigned long long path = 0;
  for (int at = last; at >= 0; at = spar[at]) path |= 1ull << at;

  const auto token = [&](int node, int row) {
    float kr[RPL];
#pragma unroll
    for (int r = 0; r < RPL; r += 8)
      unpack8(*reinterpret_cast<const uint4*>(&sk[row][rl * RPL + r]), kr + r);
    float ss = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < RPL; ++r) {
      ss = fmaf(kr[r], kr[r], ss);
      a.x = fmaf(s[r].x, kr[r], a.x);
      a.y = fmaf(s[r].y, kr[r], a.y);
      a.z = fmaf(s[r].z, kr[r], a.z);
      a.w = fmaf(s[r].w, kr[r], a.w);
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      a.x += __shfl_xor_sync(0xffffffffu, a.x, o);
      a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
      a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
      a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
    }
    const float nk = rsqrtf(ss + 1e-6f);
    const float eg = expf(sg[node]), bt = sbeta[node] * nk, en = eg * nk;
    const uint2 vu = *reinterpret_cast<const uint2*>(&sv[row][c]);
    const float4 d = make_float4(bt * (__uint_as_float(vu.x << 16) - en * a.x),
                                 bt * (__uint_as_float(vu.x & 0xffff0000u) - en * a.y),
                                 bt * (__uint_as_float(vu.y << 16) - en * a.z),
                                 bt * (__uint_as_float(vu.y & 0xffff0000u) - en * a.w));
#pragma unroll
    for (int r = 0; r < RPL; ++r) {
      s[r].x = fmaf(kr[r], d.x, s[r].x * eg);
      s[r].y = fmaf(kr[r], d.y, s[r].y * eg);
      s[r].z = fmaf(kr[r], d.z, s[r].z * eg);
      s[r].w = fmaf(kr[r], d.w, s[r].w * eg);
    }
  };
  if (n <= kStaged) {
    for (; path; path &= path - 1) {
      const int node = __ffsll(path) - 1;
      token(node, node);
    }
  } else {
    while (path) {
      const int m = min(kStaged, __popcll(path));
      stage(m, [&](int r) {
        unsigned long long p = path;
        for (int i = 0; i < r; ++i) p &= p - 1;
        return __ffsll(p) - 1;
      });
      tc::cp_async_commit();
      tc::cp_async_wait<0>();
      __syncthreads();
      for (int r = 0; r < m; ++r, path &= path - 1) token(__ffsll(path) - 1, r);
      __syncthreads();                               // the staging buffers are free
    }
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
  const bool cvec = channels % 8 == 0 && x_row_stride % 8 == 0 && conv_slot_stride % 8 == 0 &&
                    aligned16(x) && aligned16(conv_pool);
  const bool vec = k_row_stride % 8 == 0 && v_row_stride % 8 == 0 && aligned16(k) && aligned16(v);
  const int per_cta = head_v_dim * 2 * (cvec ? 8 : 1);
  const CommitConv conv{(const bf16*)x, x_row_stride, (bf16*)conv_pool, conv_slot_stride, channels,
                        kernel, (channels + per_cta - 1) / per_cta, cvec};
  const int64_t ctas = (int64_t)n_seqs * (num_v_heads + conv.ctas);
  GDN_UNSUPPORTED(ctas < (1ll << 31), "%s: too many (sequence, head) units", fn);
  cudaStream_t s = (cudaStream_t)stream;
#define GDN_CM(D)                                                                                \
  commit_tree_kernel<D, D><<<(unsigned)ctas, 2 * D, 0, s>>>(                                     \
      (const bf16*)k, k_row_stride, (const bf16*)v, v_row_stride, g, (const bf16*)beta, s_pool,  \
      slot_stride, num_slots, ids, cu_seqlens, parents, accepted, max_nodes, n_tokens, n_seqs,   \
      num_k_heads, num_v_heads, vec, conv, status)
  if (head_v_dim == 128) GDN_CM(128);
  else GDN_CM(64);
#undef GDN_CM
  return check_launch(fn);
}
