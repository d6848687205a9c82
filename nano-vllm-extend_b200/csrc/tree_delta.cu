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
// Products are computed transposed, X^T = S_0^T [K; Q]^T with mma.sync: value
// columns by 8 nodes, so few nodes waste little.  The results' layout is that of the
// next product's A operand (nodes 2t, 2t + 1 as its k = t, t + 4), so X, d and o
// never leave the warp's registers.  X is bf16 with fp32 sums: q and k are
// exact, S_0 enters as two parts of 8 bits each; A, M and d meet in tf32, two parts
// of 11 bits each (hi hi + lo hi + hi lo).  Norms, decays and the substitution
// within eight nodes are fp32.
//
// The chain of a unit (one sequence and v-head) is long and mostly latency:
// norms, decays, gram factors, X, substitution, norm.  So the states come by TMA
// (32-column boxes, 128-byte swizzle, which the fragment loads read without bank
// conflicts) into a ring of ST buffers of a persistent CTA, independent of where
// the arithmetic stands, and GROUPS groups of warps take the CTA's units in turn,
// each a whole unit.  A buffer is refilled as soon as its group has formed X.  The
// next unit's rows and scalars are loaded into registers a unit ahead.  Measured, 256
// sequences x 32 heads of 3 to 8 nodes: state loaded into registers by its own CTA,
// two CTAs an SM, 160-228 us (the loads stand still while a CTA computes); ring with
// two groups of eight warps 174 us (1000 instructions per warp and unit, most of them
// the same in every warp).  Hence few warps per unit, with 32 columns each.
//
// A node whose own d is not finite (a NaN or infinity in its row) must not reach
// nodes that do not descend from it: zero coefficients would still turn it into
// NaN, so its d is set to zero for the products and its own and its descendants'
// outputs are set to NaN at the end.
#include "mma_util.cuh"
#include "tc_util.cuh"
#include "tmap.cuh"
#include "tree.cuh"

namespace gdn {

constexpr uint32_t kDeltaWait = 1u << 22;   // polls; a state's copy takes a few microseconds

template <int D, int TN>
struct TreeDelta {
  // 16-column tiles per warp, warps and threads of a group; as many groups and
  // buffers as registers and shared memory hold
  static constexpr int MT = TN <= 32 ? 2 : 1;
  static constexpr int VC = 2 * MT;                  // value columns of a thread, adjacent
  static constexpr int NW = D / (16 * MT), NT = 32 * NW;
  static constexpr int GROUPS = TN <= 8 ? (D == 64 ? 4 : 3) : TN <= 16 ? (D == 64 ? 4 : 2) : TN <= 32 ? 2 : 1;
  static constexpr int ST = TN <= 32 ? GROUPS : 2;
  // A buffer always serves the same group: when a group waits for a unit's state it
  // has used up the buffer's last one itself, so the parity it waits for is never
  // that of two copies ago.
  static_assert(ST % GROUPS == 0, "a buffer belongs to one group");
  static constexpr bool AHEAD = TN <= 8;             // rows loaded a unit ahead
  static constexpr int KP = D + 16;                  // pitches: conflict-free fragment loads
  static constexpr int AP = TN + 4;
  static constexpr int MP = TN == 8 ? 8 : TN + 8;
  struct Group {
    __align__(16) bf16 kq[2 * TN][KP];               // keys, then queries (k order: see frag)
    float at[TN][AP];                                // at[i][j] = -A_ji
    float m[TN][MP];                                 // M
    float dec[TN][TN + 1];                           // D_ij, zero where j is no ancestor of i
    float d0[TN], eg[TN], beta[TN];
    float norm[2 * TN];                              // 1 / |k|, scale / |q|
    __align__(16) float ssum[TN][NW];
    int par[2][TN];                                  // alternating: slow warps may still walk the last unit's
  };
  struct Smem {
    __align__(1024) unsigned char state[ST][D * D * 4];
    Group group[GROUPS];
    __align__(8) unsigned long long full[ST];
  };
};

// Eight elements of a head row (vec: 16-byte aligned).
__device__ __forceinline__ uint4 load8(const bf16* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint4 u;
  bf16* h = reinterpret_cast<bf16*>(&u);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = p[e];
  return u;
}

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// (x, y) as bf16 pairs, hi + lo, both cut: 16 bits of each.
__device__ __forceinline__ void cut2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  lo = __byte_perm(__float_as_uint(x - __uint_as_float(__float_as_uint(x) & 0xffff0000u)),
                   __float_as_uint(y - __uint_as_float(__float_as_uint(y) & 0xffff0000u)), 0x7632);
}

// Substitution within eight nodes (lane t of a quad holds nodes 2t, 2t + 1; r[0],
// r[1] of one column, r[2], r[3] of the next): node i's d to the quad, then into the
// later nodes.  at: the block's -A_ji, a row per i.
template <int MT, int AP>
__device__ __forceinline__ void solve8(float (&r)[MT][4], const float* at, int lane) {
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const int e = i & 1, from = (lane & ~3) | (i >> 1);
    const float2 a = *reinterpret_cast<const float2*>(at + i * AP + 2 * (lane & 3));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const float x = __shfl_sync(0xffffffffu, r[mt][e], from);
      const float y = __shfl_sync(0xffffffffu, r[mt][2 + e], from);
      r[mt][0] = fmaf(a.x, x, r[mt][0]);
      r[mt][1] = fmaf(a.y, x, r[mt][1]);
      r[mt][2] = fmaf(a.x, y, r[mt][2]);
      r[mt][3] = fmaf(a.y, y, r[mt][3]);
    }
  }
}

// The same with nodes taken out whose d is not finite; returns them as bits.
template <int AP>
__device__ __noinline__ unsigned solve8_guarded(float4& s, const float* at, int lane) {
  unsigned bad = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const int from = (lane & ~3) | (i >> 1);
    float x = __shfl_sync(0xffffffffu, i & 1 ? s.y : s.x, from);
    float y = __shfl_sync(0xffffffffu, i & 1 ? s.w : s.z, from);
    if (!(fabsf(x) <= 3.0e38f && fabsf(y) <= 3.0e38f)) {
      bad |= 1u << i;
      x = y = 0.f;
      if (lane == from) {
        if (i & 1) s.y = s.w = 0.f;
        else s.x = s.z = 0.f;
      }
    }
    const float2 a = *reinterpret_cast<const float2*>(at + i * AP + 2 * (lane & 3));
    s.x = fmaf(a.x, x, s.x);
    s.y = fmaf(a.y, x, s.y);
    s.z = fmaf(a.x, y, s.z);
    s.w = fmaf(a.y, y, s.w);
  }
  return bad;
}

struct DeltaArgs {
  const bf16 *q, *k, *v;
  int64_t qs, ks, vs;
  const float* g;
  const bf16* beta;
  int64_t num_slots;
  const int64_t* ids;
  const int32_t* cu;
  const int32_t* parents;
  int max_nodes;
  int64_t n_tokens;
  bf16* out;
  int HK, HV, units;
  float scale;
  const bf16* z;
  int64_t zs;
  const bf16* nw;
  float eps;
  bool vec;
  int32_t* status;
};

// Where a unit is: its sequence and v-head, stepped without divisions.
struct DeltaAt {
  int seq, h;
  __device__ __forceinline__ DeltaAt step(int n, int HV) const {
    DeltaAt d{seq, h + n};
    while (d.h >= HV) {
      d.h -= HV;
      ++d.seq;
    }
    return d;
  }
};

// What it is made of, as loaded: looked at later, so that the loads can be under way.
struct DeltaRaw {
  int c0, c1;
  int64_t slot;
};

// A unit's rows and slot; n = 0: nothing to compute.
struct DeltaUnit {
  int64_t start, slot;
  int n, h;
};

template <int D, int TN, bool NORM>
__global__ void __launch_bounds__(TreeDelta<D, TN>::NT* TreeDelta<D, TN>::GROUPS, D == 64 ? 2 : 1)
    tree_delta_kernel(const __grid_constant__ CUtensorMap pool, const DeltaArgs a) {
  using P = TreeDelta<D, TN>;
  constexpr int NT = P::NT, NW = P::NW, ST = P::ST, GROUPS = P::GROUPS, MT = P::MT, VC = P::VC;
  constexpr int KB = D / 16, KT = TN / 8;
  constexpr int PC = D / 8, PPT = 2 * TN * PC / NT;   // 16-byte pieces of q / k per thread
  // gram tiles of 16 rows x 8 columns that hold a column <= some row, per half (keys, queries)
  constexpr int MH = TN / 16, TH = MH * (MH + 1), GT = TN == 8 ? 1 : (2 * TH + NW - 1) / NW;
  static_assert(2 * TN * PC % NT == 0 && TN <= NT, "thread layout");
  extern __shared__ unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<typename P::Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);

  const int group = threadIdx.x / NT, tid = threadIdx.x - group * NT;
  const int warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  typename P::Group& gs = sm.group[group];
  const auto group_sync = [&]() {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(NT) : "memory");
  };
  // this CTA's units: a run of them, group g taking every GROUPS-th
  const int u0 = (int)((int64_t)a.units * blockIdx.x / gridDim.x);
  const int count = (int)((int64_t)a.units * (blockIdx.x + 1) / gridDim.x) - u0;
  const DeltaAt first{u0 / a.HV, u0 % a.HV};
  const int last_seq = (a.units - 1) / a.HV;
  const auto raw_of = [&](const DeltaAt& at) {
    const int s = min(at.seq, last_seq);              // past the end: loaded, not used
    return DeltaRaw{a.cu[s], a.cu[s + 1], a.ids[s]};
  };
  // the i-th unit of the CTA from what was loaded for it
  const auto unit_of = [&](int i, const DeltaAt& at, const DeltaRaw& r, int32_t* status) {
    DeltaUnit d{r.c0, r.slot, 0, at.h};
    const int64_t len = (int64_t)r.c1 - r.c0;
    if (i >= count) return d;
    if (r.c0 < 0 || len < 0 || len > a.max_nodes || r.c1 > a.n_tokens) {
      if (status) atomicOr(status, GDN_STATUS_BAD_SEQLEN);
    } else if (len > 0 && slot_ok(r.slot, a.num_slots, status)) {
      d.n = (int)len;
    }
    return d;
  };
  // the state of the CTA's i-th unit into its buffer (one thread)
  const auto fetch = [&](int i, const DeltaAt& at, const DeltaRaw& r) {
    if (i >= count) return;
    const DeltaUnit d = unit_of(i, at, r, nullptr);
    const uint32_t bar = tc::smem_u32(&sm.full[i % ST]);
    if (d.n == 0) {
      tc::mbar_arrive(bar);
      return;
    }
    tc::mbar_expect_tx(bar, D * D * 4);
    const uint32_t dst = tc::smem_u32(&sm.state[i % ST][0]);
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
      tc::tma_load_3d(dst + b * D * 128, &pool, b * 32, d.h * D, (int)d.slot, bar);
  };
  if (threadIdx.x == 0) {
    for (int b = 0; b < ST; ++b) tc::mbar_init(tc::smem_u32(&sm.full[b]), 1);
    tc::mbar_init_fence();
  }
  if (threadIdx.x == NT - 1)
    asm volatile("prefetch.tensormap [%0];" ::"l"(&pool) : "memory");
  DeltaAt at_cur = first.step(group, a.HV), at_nxt = at_cur.step(GROUPS, a.HV);
  const DeltaRaw raw_cur = raw_of(at_cur), raw_nxt = raw_of(at_nxt);
  __syncthreads();
  if (tid == 0) {
    fetch(group, at_cur, raw_cur);
    for (int i = group + GROUPS; i < ST; i += GROUPS) {
      const DeltaAt at = first.step(i, a.HV);
      fetch(i, at, raw_of(at));
    }
  }

  // a unit's rows and scalars, loaded ahead
  uint4 piece[PPT];
  int my_par = -1;
  float my_g = 0.f, my_beta = 0.f;
  uint32_t vr[KT][2][MT], zr[KT][2][MT];
  const int c = warp * 16 * MT + VC * gr;            // this thread's value columns: c .. c + VC - 1
  const auto load_rows = [&](const DeltaUnit& d) {
    const int hk = d.h / (a.HV / a.HK);
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      const int p = tid + i * NT, row = p / PC, node = row % TN, ch = (p - row * PC) * 8;
      piece[i] = make_uint4(0, 0, 0, 0);
      if (node < d.n)
        piece[i] = load8((row < TN ? a.k + (d.start + node) * a.ks : a.q + (d.start + node) * a.qs) +
                             (int64_t)hk * D + ch, a.vec);
    }
    if (tid < d.n) {
      my_par = a.parents[d.start + tid];
      my_g = a.g[(d.start + tid) * a.HV + d.h];
      my_beta = bf2f(a.beta[(d.start + tid) * a.HV + d.h]);
    }
  };
  const auto load_vals = [&](uint32_t (&r)[KT][2][MT], const bf16* p, int64_t stride,
                             const DeltaUnit& d) {
    const bf16* base = p + d.start * stride + (int64_t)d.h * D + c;
#pragma unroll
    for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int node = t8 * 8 + 2 * tq + e;
        const bool on = node < d.n;
        if constexpr (MT == 2) {
          uint2 u = make_uint2(0u, 0u);
          if (on) u = *reinterpret_cast<const uint2*>(base + node * stride);
          r[t8][e][0] = u.x;
          r[t8][e][1] = u.y;
        } else {
          r[t8][e][0] = on ? *reinterpret_cast<const uint32_t*>(base + node * stride) : 0u;
        }
      }
  };
  // k-elements of row r, block kb, as this lane's fragments take them (k 2t, 2t + 1
  // and 2t + 8, 2t + 9): in shared memory those four of each 16 are adjacent
  const auto frag = [&](int r, int kb) {
    return *reinterpret_cast<const uint2*>(&gs.kq[r][kb * 16 + 4 * tq]);
  };
  // gram tile -> first row, first column
  const auto tile_at = [&](int tile, int& row0, int& col0) {
    if constexpr (TN == 8) {
      row0 = col0 = 0;
      return tile == 0;
    } else {
      const int half = tile / TH, rem = tile - half * TH;
      int mt = 0;
      while ((mt + 1) * (mt + 2) <= rem) ++mt;
      row0 = half * TN + mt * 16;
      col0 = (rem - mt * (mt + 1)) * 8;
      return tile < 2 * TH;
    }
  };
  float nwv[VC];
#pragma unroll
  for (int e = 0; e < VC; ++e) nwv[e] = NORM ? bf2f(a.nw[c + e]) : 1.f;

  int32_t* const flags = tid == 0 ? a.status : nullptr;
  DeltaAt at_fill = at_cur.step(ST, a.HV);
  DeltaUnit cur = unit_of(group, at_cur, raw_cur, flags);
  DeltaUnit nxt = unit_of(group + GROUPS, at_nxt, raw_nxt, flags);
  if constexpr (P::AHEAD) {
    load_rows(cur);
    load_vals(vr, a.v, a.vs, cur);
    if constexpr (NORM) load_vals(zr, a.z, a.zs, cur);
  }
  for (int i = group; i < count; i += GROUPS) {
    const DeltaAt at_after = at_nxt.step(GROUPS, a.HV);
    const DeltaRaw after = raw_of(at_after), fill = raw_of(at_fill);
    const uint32_t bar = tc::smem_u32(&sm.full[i % ST]);
    const int n = cur.n;
    int* par = gs.par[(i / GROUPS) & 1];
    if (n == 0) {                                    // nothing to compute: the buffer is free at once
      if (tid == 0) {
        if (!tc::mbar_wait(bar, (i / ST) & 1, kDeltaWait) && a.status)
          atomicOr(a.status, GDN_STATUS_TIMEOUT);
        fetch(i + ST, at_fill, fill);
      }
      if constexpr (P::AHEAD) {
        load_rows(nxt);
        load_vals(vr, a.v, a.vs, nxt);
        if constexpr (NORM) load_vals(zr, a.z, a.zs, nxt);
      }
    } else {
      if constexpr (!P::AHEAD) load_rows(cur);
      // q / k rows to shared memory (zero rows behind the last node) and their norms
#pragma unroll
      for (int j = 0; j < PPT; ++j) {
        const int p = tid + j * NT, row = p / PC, pc = p - row * PC;
        float f[8], ss = 0.f;
        unpack8(piece[j], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
        for (int o = PC / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (pc == 0) gs.norm[row] = rsqrtf(ss + 1e-6f) * (row < TN ? 1.f : a.scale);
        // elements 2t, 2t + 1 of the piece go to place 4t (first half of 16) or 4t + 2
        bf16* dst = &gs.kq[row][(pc >> 1) * 16 + (pc & 1) * 2];
        *reinterpret_cast<uint32_t*>(dst) = piece[j].x;
        *reinterpret_cast<uint32_t*>(dst + 4) = piece[j].y;
        *reinterpret_cast<uint32_t*>(dst + 8) = piece[j].z;
        *reinterpret_cast<uint32_t*>(dst + 12) = piece[j].w;
      }
      for (int j = tid; j < TN * (TN + 1); j += NT) (&gs.dec[0][0])[j] = 0.f;
      if (tid < TN) {
        const bool on = tid < n;
        par[tid] = on ? tree_parent(my_par, tid, a.status) : -1;
        gs.eg[tid] = on ? expf(my_g) : 0.f;
        gs.beta[tid] = on ? my_beta : 0.f;
      }
      if constexpr (P::AHEAD) load_rows(nxt);
      else load_vals(vr, a.v, a.vs, cur);
      group_sync();

      // decays: thread j walks from node j to the root
      if (tid < TN) {
        float d = 1.f;
        if (tid < n)
          for (int j = tid; j >= 0;) {
            const int up = par[j];
            const float e = gs.eg[j];
            gs.dec[tid][j] = d;
            d *= e;
            j = up;
          }
        gs.d0[tid] = tid < n ? d : 0.f;
      }
      // gram tiles [K; Q] K^T, the last warps first: the first ones walk the trees
      float gram[GT][4];
#pragma unroll
      for (int j = 0; j < GT; ++j) {
        int row0, col0;
#pragma unroll
        for (int e = 0; e < 4; ++e) gram[j][e] = 0.f;
        if (tile_at(NW - 1 - warp + j * NW, row0, col0)) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const uint2 fa = frag(row0 + gr, kb), fb = frag(row0 + gr + 8, kb), fc = frag(col0 + gr, kb);
            const uint32_t fr[4] = {fa.x, fb.x, fa.y, fb.y};
            mm::mma16816(gram[j], fr, fc.x, fc.y);
          }
        }
      }

      // X^T = S_0^T [K; Q]^T
      if (!tc::mbar_wait(bar, (i / ST) & 1, kDeltaWait)) {
        if (a.status) atomicOr(a.status, GDN_STATUS_TIMEOUT);
        tc::mbar_wait(bar, (i / ST) & 1, kDeltaWait);
      }
      float acc[2 * KT][MT][4];
#pragma unroll
      for (int t8 = 0; t8 < 2 * KT; ++t8)
#pragma unroll
        for (int e = 0; e < 4 * MT; ++e) acc[t8][e / 4][e % 4] = 0.f;
      {
        // rows 2t and 2t + 1 (mod 8: their swizzle) of every eight; a thread's columns
        // are one 16-byte piece, or half of one
        const unsigned char* box = &sm.state[i % ST][(c >> 5) * D * 128];
        const int chunk = (c & 31) >> 2, sub = (c & 3) * 4;
        const unsigned char* p0 = box + 2 * tq * 128 + ((chunk ^ (2 * tq)) << 4) + sub;
        const unsigned char* p1 = box + (2 * tq + 1) * 128 + ((chunk ^ (2 * tq + 1)) << 4) + sub;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          float s[4][VC];                            // rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned char* p = (j & 1 ? p1 : p0) + kb * 2048 + (j >> 1) * 1024;
            if constexpr (VC == 4) *reinterpret_cast<float4*>(s[j]) = *reinterpret_cast<const float4*>(p);
            else *reinterpret_cast<float2*>(s[j]) = *reinterpret_cast<const float2*>(p);
          }
          uint32_t hi[MT][4], lo[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              cut2(s[(e >> 1) * 2][2 * mt + (e & 1)], s[(e >> 1) * 2 + 1][2 * mt + (e & 1)], hi[mt][e],
                   lo[mt][e]);
#pragma unroll
          for (int t8 = 0; t8 < 2 * KT; ++t8) {
            const uint2 b = frag(t8 * 8 + gr, kb);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mm::mma16816(acc[t8][mt], hi[mt], b.x, b.y);
              mm::mma16816(acc[t8][mt], lo[mt], b.x, b.y);
            }
          }
        }
      }
      if constexpr (!P::AHEAD && NORM) load_vals(zr, a.z, a.zs, cur);
      group_sync();                                  // decays complete, the buffer is free
      if (tid == 0) fetch(i + ST, at_fill, fill);

      // gram tiles -> the factors -A and M
#pragma unroll
      for (int j = 0; j < GT; ++j) {
        int row0, col0;
        if (tile_at(NW - 1 - warp + j * NW, row0, col0)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = row0 + gr + (e >> 1) * 8, ci = col0 + 2 * tq + (e & 1), node = row % TN;
            const float d = gs.dec[node][ci];
            const float f = d == 0.f ? 0.f : d * gs.norm[ci] * gs.norm[row] * gram[j][e];
            if (row < TN) gs.at[ci][node] = ci < node ? -gs.beta[node] * f : 0.f;
            else gs.m[node][ci] = f;
          }
        }
      }
      // right sides (keys) and the state's part of the outputs (queries)
#pragma unroll
      for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int node = t8 * 8 + 2 * tq + e;
          const float b = gs.beta[node], f = gs.d0[node];
          const float fk = f * gs.norm[node], fq = f * gs.norm[TN + node];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float &k0 = acc[t8][mt][e], &k1 = acc[t8][mt][2 + e];
            k0 = node < n ? b * (bf_lo(vr[t8][e][mt]) - fk * k0) : 0.f;
            k1 = node < n ? b * (bf_hi(vr[t8][e][mt]) - fk * k1) : 0.f;
            acc[KT + t8][mt][e] *= fq;
            acc[KT + t8][mt][2 + e] *= fq;
          }
        }
      if constexpr (P::AHEAD) load_vals(vr, a.v, a.vs, nxt);
      group_sync();                                  // the factors are complete

      unsigned long long bad = 0;
#pragma unroll
      for (int blk = 0; blk < KT; ++blk) {
        if (blk * 8 < n) {
          float(&r)[MT][4] = acc[blk];
          float s[MT][4], size = 0.f;
#pragma unroll
          for (int e = 0; e < 4 * MT; ++e) s[e / 4][e % 4] = r[e / 4][e % 4];
          solve8<MT, P::AP>(r, &gs.at[blk * 8][blk * 8], lane);
#pragma unroll
          for (int e = 0; e < 4 * MT; ++e) size += fabsf(r[e / 4][e % 4]);
          // not finite where a part is not (or where the sum ran over)
          if (__any_sync(0xffffffffu, !(size <= 3.0e38f))) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float4 t = make_float4(s[mt][0], s[mt][1], s[mt][2], s[mt][3]);
              bad |= (unsigned long long)solve8_guarded<P::AP>(t, &gs.at[blk * 8][blk * 8], lane)
                     << (blk * 8);
              r[mt][0] = t.x;
              r[mt][1] = t.y;
              r[mt][2] = t.z;
              r[mt][3] = t.w;
            }
          }
          // this block's d as an A operand, into the later blocks and the outputs
          uint32_t hi[MT][4], lo[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mm::split_tf32(r[mt][0], hi[mt][0], lo[mt][0]);
            mm::split_tf32(r[mt][2], hi[mt][1], lo[mt][1]);
            mm::split_tf32(r[mt][1], hi[mt][2], lo[mt][2]);
            mm::split_tf32(r[mt][3], hi[mt][3], lo[mt][3]);
          }
          const auto add = [&](float(&to)[MT][4], float f0, float f1) {
            uint32_t h0, l0, h1, l1;
            mm::split_tf32(f0, h0, l0);
            mm::split_tf32(f1, h1, l1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mm::mma1688(to[mt], hi[mt][0], hi[mt][1], hi[mt][2], hi[mt][3], h0, h1);
              mm::mma1688(to[mt], lo[mt][0], lo[mt][1], lo[mt][2], lo[mt][3], h0, h1);
              mm::mma1688(to[mt], hi[mt][0], hi[mt][1], hi[mt][2], hi[mt][3], l0, l1);
            }
          };
#pragma unroll
          for (int t8 = blk + 1; t8 < KT; ++t8)
            add(acc[t8], gs.at[blk * 8 + 2 * tq][t8 * 8 + gr], gs.at[blk * 8 + 2 * tq + 1][t8 * 8 + gr]);
#pragma unroll
          for (int t8 = blk; t8 < KT; ++t8) {
            const float2 f = *reinterpret_cast<const float2*>(&gs.m[t8 * 8 + gr][blk * 8 + 2 * tq]);
            add(acc[KT + t8], f.x, f.y);
          }
        }
      }
      if (__any_sync(0xffffffffu, bad != 0)) {
        bad = (unsigned long long)__reduce_or_sync(0xffffffffu, (unsigned)(bad >> 32)) << 32 |
              __reduce_or_sync(0xffffffffu, (unsigned)bad);
#pragma unroll
        for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            for (int j = t8 * 8 + 2 * tq + e; j >= 0; j = par[j])
              if (bad >> j & 1) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                  acc[KT + t8][mt][e] = acc[KT + t8][mt][2 + e] = __int_as_float(0x7fffffff);
                break;
              }
      }

      if constexpr (NORM) {
#pragma unroll
        for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float ss = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              ss = fmaf(acc[KT + t8][mt][e], acc[KT + t8][mt][e], ss);
              ss = fmaf(acc[KT + t8][mt][2 + e], acc[KT + t8][mt][2 + e], ss);
            }
            ss += __shfl_xor_sync(0xffffffffu, ss, 4);
            ss += __shfl_xor_sync(0xffffffffu, ss, 8);
            ss += __shfl_xor_sync(0xffffffffu, ss, 16);
            if (gr == 0) gs.ssum[t8 * 8 + 2 * tq + e][warp] = ss;
          }
        group_sync();
      }
      bf16* obase = a.out + (cur.start * a.HV + cur.h) * D + c;
#pragma unroll
      for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int node = t8 * 8 + 2 * tq + e;
          if (node >= n) continue;
          float o[VC];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            o[2 * mt] = acc[KT + t8][mt][e];
            o[2 * mt + 1] = acc[KT + t8][mt][2 + e];
          }
          if constexpr (NORM) {
            float tot = 0.f;
#pragma unroll
            for (int j = 0; j < NW; ++j) tot += gs.ssum[node][j];
            const float inv = rsqrtf(tot * (1.f / D) + a.eps);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              o[2 * mt] *= inv * nwv[2 * mt] * conv_silu(bf_lo(zr[t8][e][mt]));
              o[2 * mt + 1] *= inv * nwv[2 * mt + 1] * conv_silu(bf_hi(zr[t8][e][mt]));
            }
          }
          bf16* to = obase + (int64_t)node * a.HV * D;
          if constexpr (MT == 2)
            *reinterpret_cast<uint2*>(to) = make_uint2(mm::pack2(o[0], o[1]), mm::pack2(o[2], o[3]));
          else
            *reinterpret_cast<uint32_t*>(to) = mm::pack2(o[0], o[1]);
        }
      if constexpr (P::AHEAD && NORM) load_vals(zr, a.z, a.zs, nxt);
    }
    cur = nxt;
    nxt = unit_of(i + 2 * GROUPS, at_after, after, flags);
    at_nxt = at_after;
    at_fill = at_fill.step(GROUPS, a.HV);
  }
}

template <int D, int TN>
static int launch_tree_delta(const CUtensorMap& pool, const DeltaArgs& a, cudaStream_t s) {
  using P = TreeDelta<D, TN>;
  constexpr size_t bytes = sizeof(typename P::Smem) + 1024;
  static_assert(bytes <= 227 * 1024, "shared memory of one SM");
  auto fn = a.z != nullptr ? tree_delta_kernel<D, TN, true> : tree_delta_kernel<D, TN, false>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
      cudaSuccess)
    return check_launch("gdn_delta_rule_tree");
  // persistent: as many CTAs as fit the SMs at once
  const int fit = D == 64 && 2 * bytes <= 227 * 1024 ? 2 : 1;
  const int64_t most = (int64_t)sm_count() * fit;
  fn<<<(unsigned)(a.units < most ? a.units : most), P::NT * P::GROUPS, bytes, s>>>(pool, a);
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
  GDN_UNSUPPORTED(v_row_stride % 4 == 0 && (z == nullptr || z_row_stride % 4 == 0) &&
                      ((uintptr_t)v | (uintptr_t)z | (uintptr_t)out) % 8 == 0,
                  "%s: v, z and out must be 8-byte aligned with row strides of whole fours", fn);
  const int64_t units = (int64_t)n_seqs * num_v_heads;
  GDN_UNSUPPORTED(units < (1ll << 30), "%s: too many (sequence, head) units", fn);
  // the pool's view as rows of value columns, [slots][HV * DK][DV]
  const EncodeTiledFn encode = encode_tiled();
  const cuuint64_t dims[3] = {(cuuint64_t)head_v_dim, (cuuint64_t)num_v_heads * head_k_dim,
                              (cuuint64_t)num_slots};
  const cuuint64_t strides[2] = {(cuuint64_t)head_v_dim * 4, (cuuint64_t)slot_stride * 4};
  const cuuint32_t box[3] = {32, (cuuint32_t)head_k_dim, 1}, step[3] = {1, 1, 1};
  CUtensorMap pool;
  GDN_UNSUPPORTED(num_slots < (1ll << 31), "%s: too many slots", fn);
  if (encode == nullptr ||
      encode(&pool, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(s_pool), dims, strides,
             box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    set_error("%s: the pool's tensor map could not be encoded", fn);
    return GDN_ERR_CUDA;
  }
  const DeltaArgs a{(const bf16*)q, (const bf16*)k, (const bf16*)v, q_row_stride, k_row_stride,
                    v_row_stride, g, (const bf16*)beta, num_slots, ids, cu_seqlens, parents,
                    max_nodes, n_tokens, (bf16*)out, num_k_heads, num_v_heads, (int)units, scale,
                    (const bf16*)z, z_row_stride, (const bf16*)norm_weight, norm_eps,
                    aligned16(q) && aligned16(k) && q_row_stride % 8 == 0 && k_row_stride % 8 == 0,
                    status};
  cudaStream_t s = (cudaStream_t)stream;
#define GDN_TDN(D)                                             \
  if (max_nodes <= 8) return launch_tree_delta<D, 8>(pool, a, s);   \
  if (max_nodes <= 16) return launch_tree_delta<D, 16>(pool, a, s); \
  if (max_nodes <= 32) return launch_tree_delta<D, 32>(pool, a, s); \
  return launch_tree_delta<D, 64>(pool, a, s)
  if (head_v_dim == 128) { GDN_TDN(128); }
  GDN_TDN(64);
#undef GDN_TDN
}
