// Query / key head norms, the position rotation and the paged-cache store in
// one pass over the rows of the attention layer's projection.
//
//   x^ = x * rsqrt(mean(x^2) + eps) * w      (or * (1 + w): unit_offset)
//   y[i]       = x^[i] cos_p[i] - x^[i + R/2] sin_p[i]        i < R/2
//   y[i + R/2] = x^[i + R/2] cos_p[i] + x^[i] sin_p[i];       y[i] = x^[i], i >= R
// for every query and key head, p the row's position and R = rot; keys and
// values go to their row's cache slot (-1: nowhere), queries to q_out.
//
// HBM-bound: every element is read once and written once (4 bytes), the table of
// cosines and sines is R * 4 bytes per row, shared by the row's heads in L1 / L2.
// D / 8 lanes own one head of one row, 16 bytes each; the norm is a shuffle sum
// and the rotation's partner half comes from the lane R / 16 away, so nothing
// goes through shared memory.  All arithmetic is fp32, rounded once at the end.
#include "tree.cuh"

namespace gdn {

constexpr int kRopeThreads = 256;

template <int D>
__global__ void __launch_bounds__(kRopeThreads) qk_rope_kernel(
    const bf16* __restrict__ q, int64_t qs, const bf16* __restrict__ k, int64_t ks,
    const bf16* __restrict__ v, int64_t vs, const bf16* __restrict__ qw,
    const bf16* __restrict__ kw, float eps, float offset, const float* __restrict__ cos_sin,
    int64_t max_pos, int rot, const int64_t* __restrict__ positions, bf16* __restrict__ k_cache,
    bf16* __restrict__ v_cache, int64_t block_stride, int64_t token_stride, int64_t head_stride,
    int64_t num_blocks, int block_size, const int32_t* __restrict__ slots, bf16* __restrict__ out,
    int64_t n_tokens, int HQ, int HKV, int32_t* status) {
  constexpr int LPR = D / 8;                  // lanes per head
  const int heads = HQ + 2 * HKV;
  const int64_t item = ((int64_t)blockIdx.x * kRopeThreads + threadIdx.x) / LPR;
  const bool live = item < n_tokens * heads;
  const int64_t t = live ? item / heads : 0;
  const int h = live ? (int)(item - t * heads) : 0;
  const int sub = threadIdx.x % LPR;
  const int d0 = sub * 8;

  const bool is_q = h < HQ, is_v = h >= HQ + HKV;
  const int kvh = is_q ? 0 : is_v ? h - HQ - HKV : h - HQ;
  const bf16* src = is_q ? q + t * qs + (int64_t)h * D
                         : is_v ? v + t * vs + (int64_t)kvh * D : k + t * ks + (int64_t)kvh * D;
  const uint4 raw = live ? *reinterpret_cast<const uint4*>(src + d0) : make_uint4(0, 0, 0, 0);
  int64_t pos = 0;
  bool ok = live;
  if (live && !is_v) {
    pos = positions[t];
    if (pos < 0 || pos >= max_pos) {
      if (status && sub == 0) atomicOr(status, GDN_STATUS_BAD_POSITION);
      ok = false;
      pos = 0;
    }
  }
  bf16* dst = nullptr;
  if (live && is_q) {
    dst = out + (t * HQ + h) * D;
  } else if (live) {
    const int64_t slot = slots[t];
    if (slot >= 0 && slot < num_blocks * block_size) {
      const int64_t page = slot / block_size;
      dst = (is_v ? v_cache : k_cache) + page * block_stride +
            (slot - page * block_size) * token_stride + (int64_t)kvh * head_stride;
    } else if (slot != -1) {
      if (status && sub == 0) atomicOr(status, GDN_STATUS_BAD_SLOT);
    }
  }
  float x[8];
  unpack8(raw, x);
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(ss * (1.f / D) + eps);
  float wv[8];
  unpack8(*reinterpret_cast<const uint4*>((is_q ? qw : kw) + d0), wv);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (wv[e] + offset);

  // the rotation's other half: the lane rot / 16 away, within this head's lanes
  const int half = rot / 2, far = rot / 16;
  const bool lo = d0 < half, turn = d0 < rot;
  const int lane = threadIdx.x & 31;
  const int from = turn ? (lo ? lane + far : lane - far) : lane;
  float other[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) other[e] = __shfl_sync(0xffffffffu, x[e], from);
  if (dst == nullptr || !ok) return;
  if (is_v) {
    *reinterpret_cast<uint4*>(dst + d0) = raw;
    return;
  }
  if (turn) {
    const float* cs = cos_sin + pos * rot + (lo ? d0 : d0 - half);
    float c[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(cs + e);
      *reinterpret_cast<float4*>(s + e) = *reinterpret_cast<const float4*>(cs + half + e);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * c[e] + (lo ? -other[e] : other[e]) * s[e];
  }
  *reinterpret_cast<uint4*>(dst + d0) = pack8(x);
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_qk_norm_rope_cache(
    const void* q, int64_t q_row_stride, const void* k, int64_t k_row_stride, const void* v,
    int64_t v_row_stride, const void* q_weight, const void* k_weight, float eps,
    int32_t unit_offset, const float* cos_sin, int64_t max_position, int32_t rotary_dim,
    const int64_t* positions, void* k_cache, void* v_cache, int64_t block_stride,
    int64_t token_stride, int64_t head_stride, int64_t num_blocks, int32_t block_size,
    const int32_t* slot_mapping, void* q_out, int64_t n_tokens, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t* status, void* stream) {
  clear_error();
  const char* fn = "gdn_qk_norm_rope_cache";
  GDN_REQUIRE(n_tokens >= 0 && num_q_heads > 0 && num_kv_heads > 0,
              "%s: bad sizes (n_tokens=%lld, HQ=%d, HKV=%d)", fn, (long long)n_tokens,
              num_q_heads, num_kv_heads);
  GDN_UNSUPPORTED(head_dim == 64 || head_dim == 128 || head_dim == 256,
                  "%s: head dim %d unsupported (64, 128, 256)", fn, head_dim);
  GDN_UNSUPPORTED(rotary_dim >= 16 && rotary_dim <= head_dim && rotary_dim % 16 == 0,
                  "%s: rotary dim %d unsupported (a multiple of 16 up to the head dim)", fn,
                  rotary_dim);
  GDN_REQUIRE(q_row_stride >= (int64_t)num_q_heads * head_dim &&
                  k_row_stride >= (int64_t)num_kv_heads * head_dim &&
                  v_row_stride >= (int64_t)num_kv_heads * head_dim,
              "%s: row stride smaller than the heads it holds", fn);
  GDN_REQUIRE(num_blocks >= 0 && block_size > 0 && max_position > 0,
              "%s: bad cache or table sizes", fn);
  GDN_REQUIRE(head_stride >= head_dim && token_stride >= head_dim && block_stride >= head_dim,
              "%s: cache strides smaller than a head", fn);
  if (n_tokens == 0) return GDN_OK;
  GDN_REQUIRE(q && k && v && q_weight && k_weight && cos_sin && positions && slot_mapping && q_out &&
                  ((k_cache && v_cache) || num_blocks == 0),
              "%s: null pointer", fn);
  GDN_UNSUPPORTED(((q_row_stride | k_row_stride | v_row_stride | block_stride | token_stride |
                    head_stride) & 7) == 0 &&
                      aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_weight) &&
                      aligned16(k_weight) && aligned16(cos_sin) && aligned16(q_out) &&
                      aligned16(k_cache) && aligned16(v_cache),
                  "%s: operands and strides must be 16-byte aligned", fn);
  const int64_t items = n_tokens * (num_q_heads + 2ll * num_kv_heads);
  const int64_t per_cta = kRopeThreads / (head_dim / 8);
  const int64_t ctas = (items + per_cta - 1) / per_cta;
  GDN_UNSUPPORTED(ctas < (1ll << 31), "%s: too many rows", fn);
  cudaStream_t s = (cudaStream_t)stream;
#define GDN_ROPE(DD)                                                                             \
  case DD:                                                                                       \
    qk_rope_kernel<DD><<<(unsigned)ctas, kRopeThreads, 0, s>>>(                                  \
        (const bf16*)q, q_row_stride, (const bf16*)k, k_row_stride, (const bf16*)v,              \
        v_row_stride, (const bf16*)q_weight, (const bf16*)k_weight, eps, unit_offset ? 1.f : 0.f, \
        cos_sin, max_position, rotary_dim, positions, (bf16*)k_cache, (bf16*)v_cache,            \
        block_stride, token_stride, head_stride, num_blocks, block_size, slot_mapping,           \
        (bf16*)q_out, n_tokens, num_q_heads, num_kv_heads, status);                              \
    break;
  switch (head_dim) { GDN_ROPE(64) GDN_ROPE(128) GDN_ROPE(256) }
#undef GDN_ROPE
  return check_launch(fn);
}
