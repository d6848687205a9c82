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
// D / 8 lanes own NH heads of one row, eight elements of each per lane: their loads are
// in flight together and they share the position, the slot and the table's row.  A lane's
// elements are four of the first half of the rotation and their four partners of
// the second, or eight behind it, so the rotation needs no exchange (with 16-byte
// pieces and shuffles for the partners 27 us where this takes 24).  The norm is a
// shuffle sum.  All arithmetic is fp32, rounded once at the end.
//
// NH: 6 where that many rows fill the GPU anyway (8.3k rows of 16 + 4 + 4 heads x 128:
// 1 head 35 us, 2 28, 4 26, 6 24, 8 29; floor 16), else 2, which spread a small call
// over more SMs (128 rows: 2.6 us where 6 take 4.2).  The rule does not look at the number
// of heads, and where six do not divide it lanes are without one: 8 heads (25k rows) 32.8 us
// where NH = 4 takes 27.7, 10 heads (20k) 27.2 where 5 takes 25.1, 7 heads (29k) 35.5 where 8
// takes 27.4; 12 and 24 heads are best with 6.
#include "mma_util.cuh"
#include "tree.cuh"

namespace gdn {

constexpr int kRopeThreads = 256;

template <int D, int NH>
__global__ void __launch_bounds__(kRopeThreads, 4) qk_rope_kernel(
    const bf16* __restrict__ q, int64_t qs, const bf16* __restrict__ k, int64_t ks,
    const bf16* __restrict__ v, int64_t vs, const bf16* __restrict__ qw,
    const bf16* __restrict__ kw, float eps, float offset, const float* __restrict__ cos_sin,
    int64_t max_pos, int rot, const int64_t* __restrict__ positions, bf16* __restrict__ k_cache,
    bf16* __restrict__ v_cache, int64_t block_stride, int64_t token_stride, int64_t head_stride,
    int64_t num_blocks, int block_size, const int32_t* __restrict__ slots, bf16* __restrict__ out,
    int64_t n_tokens, int HQ, int HKV, int groups, int32_t* status) {
  constexpr int LPR = D / 8;                  // lanes per head
  const int heads = HQ + 2 * HKV;
  const int64_t item = (int64_t)blockIdx.x * (kRopeThreads / LPR) + threadIdx.x / LPR;
  const bool live = item < n_tokens * groups;
  const int64_t t = live ? (item >> 31 ? item / groups : (int64_t)((unsigned)item / (unsigned)groups)) : 0;
  const int h0 = live ? (int)(item - t * groups) * NH : heads;
  // this lane's elements: da .. da + 3 and db .. db + 3
  const int sub = threadIdx.x % LPR, half = rot / 2;
  const bool turn = sub < rot / 8;
  const int da = turn ? sub * 4 : sub * 8, db = turn ? half + sub * 4 : sub * 8 + 4;

  uint2 ra[NH], rb[NH];
#pragma unroll
  for (int u = 0; u < NH; ++u) {
    const int h = h0 + u;
    ra[u] = rb[u] = make_uint2(0, 0);
    if (h < heads) {
      const bf16* src = h < HQ ? q + t * qs + (int64_t)h * D
                               : h < HQ + HKV ? k + t * ks + (int64_t)(h - HQ) * D
                                              : v + t * vs + (int64_t)(h - HQ - HKV) * D;
      ra[u] = *reinterpret_cast<const uint2*>(src + da);
      rb[u] = *reinterpret_cast<const uint2*>(src + db);
    }
  }
  int64_t pos = live ? positions[t] : 0;
  const int slot = live ? slots[t] : -1;
  const bool placed = pos >= 0 && pos < max_pos;
  if (!placed) {
    if (status && sub == 0 && h0 < HQ + HKV) atomicOr(status, GDN_STATUS_BAD_POSITION);
    pos = 0;
  }
  int64_t cache = -1;                         // the slot's place in the caches
  if (slot >= 0 && slot < num_blocks * block_size) {
    const int page = slot / block_size;
    // (a row without a position has no key: its value would stand beside an older one)
    if (placed) cache = page * block_stride + (int64_t)(slot - page * block_size) * token_stride;
  } else if (slot != -1 && status && sub == 0 && h0 + NH > HQ) {
    atomicOr(status, GDN_STATUS_BAD_SLOT);
  }
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (turn && h0 < HQ + HKV) {
    c = *reinterpret_cast<const float4*>(cos_sin + pos * rot + da);
    s = *reinterpret_cast<const float4*>(cos_sin + pos * rot + db);
  }
  const auto unpack4 = [](const uint2& u, float(&f)[4]) {
    f[0] = __uint_as_float(u.x << 16);
    f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16);
    f[3] = __uint_as_float(u.y & 0xffff0000u);
  };
  float wa[4], wb[4];                         // weights of the heads' kind
  const auto weights = [&](const bf16* w) {
    unpack4(*reinterpret_cast<const uint2*>(w + da), wa);
    unpack4(*reinterpret_cast<const uint2*>(w + db), wb);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      wa[e] += offset;
      wb[e] += offset;
    }
  };
  weights(h0 < HQ ? qw : kw);
#pragma unroll
  for (int u = 0; u < NH; ++u) {
    const int h = h0 + u;
    if (h == HQ && u > 0) weights(kw);
    float a[4], b[4];
    unpack4(ra[u], a);
    unpack4(rb[u], b);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.f / D) + eps);
    bf16* dst = nullptr;
    if (h < HQ) {
      if (placed) dst = out + (t * HQ + h) * D;
    } else if (h < heads && cache >= 0) {
      if (h >= HQ + HKV) {
        dst = v_cache + cache + (h - HQ - HKV) * head_stride;
        *reinterpret_cast<uint2*>(dst + da) = ra[u];
        *reinterpret_cast<uint2*>(dst + db) = rb[u];
        dst = nullptr;
      } else {
        dst = k_cache + cache + (h - HQ) * head_stride;
      }
    }
    if (dst != nullptr) {
      const float cc[4] = {c.x, c.y, c.z, c.w}, sc[4] = {s.x, s.y, s.z, s.w};
      float y[4], z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = a[e] * inv * wa[e], x1 = b[e] * inv * wb[e];
        y[e] = x0 * cc[e] - x1 * sc[e];
        z[e] = x1 * cc[e] + x0 * sc[e];
      }
      *reinterpret_cast<uint2*>(dst + da) = make_uint2(mm::pack2(y[0], y[1]), mm::pack2(y[2], y[3]));
      *reinterpret_cast<uint2*>(dst + db) = make_uint2(mm::pack2(z[0], z[1]), mm::pack2(z[2], z[3]));
    }
  }
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
  const int heads = num_q_heads + 2 * num_kv_heads;
  // one full wave of threads with two heads each: enough rows for six
  const bool many = n_tokens * heads * (head_dim / 8) / 2 >= (int64_t)sm_count() * 2048;
  const int nh = many ? 6 : 2, groups = (heads + nh - 1) / nh;
  const int64_t items = n_tokens * groups;
  const int64_t per_cta = kRopeThreads / (head_dim / 8);
  const int64_t ctas = (items + per_cta - 1) / per_cta;
  GDN_UNSUPPORTED(ctas < (1ll << 31), "%s: too many rows", fn);
  cudaStream_t s = (cudaStream_t)stream;
#define GDN_ROPE(DD, NH)                                                                          \
  qk_rope_kernel<DD, NH><<<(unsigned)ctas, kRopeThreads, 0, s>>>(                                 \
      (const bf16*)q, q_row_stride, (const bf16*)k, k_row_stride, (const bf16*)v, v_row_stride,   \
      (const bf16*)q_weight, (const bf16*)k_weight, eps, unit_offset ? 1.f : 0.f, cos_sin,        \
      max_position, rotary_dim, positions, (bf16*)k_cache, (bf16*)v_cache, block_stride,          \
      token_stride, head_stride, num_blocks, block_size, slot_mapping, (bf16*)q_out, n_tokens,    \
      num_q_heads, num_kv_heads, groups, status)
#define GDN_ROPE2(DD)               \
  if (head_dim == DD) {             \
    if (many) GDN_ROPE(DD, 6);      \
    else GDN_ROPE(DD, 2);           \
  }
  GDN_ROPE2(64) GDN_ROPE2(128) GDN_ROPE2(256)
#undef GDN_ROPE2
#undef GDN_ROPE
  return check_launch(fn);
}
