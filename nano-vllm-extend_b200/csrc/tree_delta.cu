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
// never leave the warp's registers.  X is bf16 with fp32 sums: q and k are exact,
// S_0 enters as two parts, each rounded: 2^-17 of an element is left out, which moves
// outputs by 5e-5 relative, where their own rounding is 1.7e-3 (all 24 bits, in three parts:
// 107 us instead of 97; one tf32 part of 11 bits saves 2 of them); A, M and d meet in
// tf32, two parts of 11 bits each (hi hi + lo hi + hi lo).  Norms, decays and the
// substitution within eight nodes are fp32.
//
// The chain of a unit (one sequence and v-head) is long and mostly latency:
// norms, decays, gram factors, X, substitution, norm.  So the states come by TMA
// (32-column boxes, 128-byte swizzle, which the fragment loads read without bank
// conflicts) into a ring of ST buffers of a persistent CTA, independent of where
// the arithmetic stands, and GROUPS groups of warps take the CTA's units in turn,
// each a whole unit.  A buffer is refilled as soon as its group has formed X.  Rows,
// values and gates of the next unit are copied into shared memory a unit ahead
// (cp.async): as loads into registers they made every other wait of the warp a wait
// for memory (a warp has six scoreboards), 115 us where this took 99.  Measured
// so, 256 sequences x 32 heads of 3 to 8 nodes, the floor being 89 us: state loaded
// into registers by its own CTA, two CTAs an SM, 160-228 us (the loads stand still
// while a CTA computes); the ring with two groups of eight warps 174 (1000
// instructions per warp and unit, most of them the same in every warp: hence few
// warps per unit, with 32 columns each).
//
// A d that is not finite (a NaN or infinity in the node's row, in the state, or past
// the largest value) must not reach nodes that do not descend from it: zero
// coefficients would still turn it into NaN, so it is set to zero for the products and
// the outputs of its node and the node's descendants are set to NaN, in its value
// column alone, as the recurrence has it.
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
  static constexpr int GROUPS = D == 64 ? (TN <= 8 ? 4 : TN <= 16 ? 3 : TN <= 32 ? 2 : 1)
                                        : (TN <= 8 ? 3 : TN <= 32 ? 2 : 1);
  static constexpr int ST = TN <= 32 ? GROUPS : 2;
  // A buffer always serves the same group: when a group waits for a unit's state it
  // has used up the buffer's last one itself, so the parity it waits for is never
  // that of two copies ago.
  static_assert(ST % GROUPS == 0, "a buffer belongs to one group");
  static constexpr bool AHEAD = TN <= 32;            // values and gates copied a unit ahead
  static constexpr int KP = D + 8;                   // pitches: conflict-free fragment loads
  static constexpr int AP = TN + 4;
  static constexpr int MP = TN == 8 ? 8 : TN + 8;
  struct Group {
    __align__(16) bf16 kq[2 * TN][KP];               // keys, then queries
    float at[TN][AP];                                // at[i][j] = -A_ji
    float m[TN][MP];                                 // M
    float dec[TN][TN + 1];                           // D_ij, zero where j is no ancestor of i
    float d0[TN], eg[TN], beta[TN];
    float norm[2 * TN];                              // 1 / |k|, scale / |q|
    __align__(16) float ssum[TN][NW];
    int lost;                                        // a state did not come in time: the group has given up
    int par[2][TN];                                  // alternating: slow warps may still walk the last unit's
    // values and gates: each thread's own pieces, [node of the thread][thread]
    __align__(16) unsigned char vals[2][AHEAD ? TN / 4 * NT * MT * 4 : 16];
  };
  struct Smem {
    __align__(1024) unsigned char state[ST][D * D * 4];
    Group group[GROUPS];
    __align__(8) unsigned long long full[ST];
  };
};

// Eight elements of an unaligned head row.
__device__ __forceinline__ uint4 load8(const bf16* p) {
  uint4 u;
  bf16* h = reinterpret_cast<bf16*>(&u);
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = p[e];
  return u;
}

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

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

// The same with what is not finite taken out; returns it as bits, the first column's
// eight nodes, then the second's.
template <int AP>
__device__ __noinline__ unsigned solve8_guarded(float4& s, const float* at, int lane) {
  unsigned bad = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const int from = (lane & ~3) | (i >> 1);
    float x = __shfl_sync(0xffffffffu, i & 1 ? s.y : s.x, from);
    float y = __shfl_sync(0xffffffffu, i & 1 ? s.w : s.z, from);
    if (!isfinite(x)) {
      bad |= 1u << i;
      x = 0.f;
      if (lane == from) (i & 1 ? s.y : s.x) = 0.f;
    }
    if (!isfinite(y)) {
      bad |= 256u << i;
      y = 0.f;
      if (lane == from) (i & 1 ? s.w : s.z) = 0.f;
    }
    const float2 a = *reinterpret_cast<const float2*>(at + i * AP + 2 * (lane & 3));
    s.x = fmaf(a.x, x, s.x);
    s.y = fmaf(a.y, x, s.y);
    s.z = fmaf(a.x, y, s.z);
    s.w = fmaf(a.y, y, s.w);
  }
  return bad;
}

// The nodes of block `blk` (of eight) on the path of `node`, as bits.
__device__ __noinline__ unsigned path_in_block(const int* par, int node, int blk) {
  unsigned on = 0;
  for (int j = node; j >= blk * 8; j = par[j])
    if (j < blk * 8 + 8) on |= 1u << (j - blk * 8);
  return on;
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
  int HV, units;
  unsigned rep_magic;   // ceil(2^32 / v-heads per k-head), so that h * it >> 32 is the k-head (h < 2^16); 0: one
  float scale;
  const bf16* z;
  int64_t zs;
  const bf16* nw;
  float eps;
  bool vec;
  uint32_t wait;        // polls for a state's copy
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
  constexpr int NPP = NT / PC;                       // rows from one piece of a thread to the next
  // gram tiles of 16 rows x 8 columns: [K; Q] K^T where some column <= some row, TH per
  // half, then the diagonal ones of Q Q^T, for the norms
  constexpr int MH = TN / 16, TH = MH * (MH + 1), TILES = TN == 8 ? 2 : 2 * TH + 2 * MH;
  constexpr int GT = (TILES + NW - 1) / NW;
  static_assert(PPT % 2 == 0 && NT % PC == 0 && 2 * TN * PC % NT == 0 && TN <= NT, "thread layout");
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
  // the state of the CTA's i-th unit into its buffer (one thread of its group)
  int asked = -1;                                    // the last unit it asked for
  const auto fetch = [&](int i, const DeltaUnit& d) {
    if (i >= count) return;
    asked = i;
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
  if (tid == 0) gs.lost = 0;
  if (threadIdx.x == NT - 1)
    asm volatile("prefetch.tensormap [%0];" ::"l"(&pool) : "memory");
  DeltaAt at_cur = first.step(group, a.HV), at_nxt = at_cur.step(GROUPS, a.HV);
  const DeltaRaw raw_cur = raw_of(at_cur), raw_nxt = raw_of(at_nxt);
  __syncthreads();
  // bounded: the state of the CTA's i-th unit has arrived, or the group gives up at its
  // next barrier
  const auto await_state = [&](int i) {
    if (tc::mbar_wait(tc::smem_u32(&sm.full[i % ST]), (i / ST) & 1, a.wait)) return;
    gs.lost = 1;
    if (a.status) atomicOr(a.status, GDN_STATUS_TIMEOUT);
  };

  // a unit's scalars, loaded ahead
  int my_par = -1;
  float my_g = 0.f, my_beta = 0.f;
  const int c = warp * 16 * MT + VC * gr;            // this thread's value columns: c .. c + VC - 1
  // q / k rows to shared memory (zero rows behind the last node), a thread's first
  // pieces keys, the others queries; and the nodes' scalars to registers
  const int node0 = tid / PC, ch = tid % PC * 8;
  const int64_t koff = node0 * a.ks + ch, qoff = node0 * a.qs + ch;
  const auto load_rows = [&](const DeltaUnit& d) {
    const int hk = a.rep_magic ? (int)__umulhi((unsigned)d.h, a.rep_magic) : d.h;
    const bf16* kp = a.k + d.start * a.ks + hk * D + koff;
    const bf16* qp = a.q + d.start * a.qs + hk * D + qoff;
#pragma unroll
    for (int i = 0; i < PPT / 2; ++i) {
      const int node = node0 + i * NPP;
      bf16 *kd = &gs.kq[node][ch], *qd = &gs.kq[TN + node][ch];
      if (a.vec) {
        const uint32_t bytes = node < d.n ? 16u : 0u;
        tc::cp_async16(tc::smem_u32(kd), bytes ? kp + i * NPP * a.ks : a.k, bytes);
        tc::cp_async16(tc::smem_u32(qd), bytes ? qp + i * NPP * a.qs : a.q, bytes);
      } else {
        uint4 u = make_uint4(0, 0, 0, 0), w = u;
        if (node < d.n) {
          u = load8(kp + i * NPP * a.ks);
          w = load8(qp + i * NPP * a.qs);
        }
        *reinterpret_cast<uint4*>(kd) = u;
        *reinterpret_cast<uint4*>(qd) = w;
      }
    }
    tc::cp_async_commit();
    if (tid < d.n) {
      const int64_t at = (d.start + tid) * a.HV + d.h;
      my_par = a.parents[d.start + tid];
      my_g = a.g[at];
      my_beta = bf2f(a.beta[at]);
    }
  };
  // values (which 0) or gates (1) of a unit: copied into the thread's own pieces of
  // shared memory (which ties up no register while it is under way), and read back; or,
  // where there is no room for that, loaded
  const auto copy_vals = [&](int which, const bf16* p, int64_t stride, const DeltaUnit& d) {
    if constexpr (P::AHEAD) {
      const bf16* base = p + d.start * stride + (int64_t)d.h * D + c;
#pragma unroll
      for (int j = 0; j < TN / 4; ++j) {
        const int node = j / 2 * 8 + 2 * tq + j % 2;
        const uint32_t dst = tc::smem_u32(&gs.vals[which][(j * NT + tid) * MT * 4]);
        const uint32_t bytes = node < d.n ? MT * 4u : 0u;
        const bf16* src = bytes ? base + node * stride : p;
        if constexpr (MT == 2)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                       : "memory");
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                       : "memory");
      }
    }
  };
  const auto load_vals = [&](uint32_t (&r)[KT][2][MT], int which, const bf16* p, int64_t stride,
                             const DeltaUnit& d) {
    const bf16* base = p + d.start * stride + (int64_t)d.h * D + c;
#pragma unroll
    for (int t8 = 0; t8 < KT; ++t8)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int node = t8 * 8 + 2 * tq + e;
        const unsigned char* src =
            P::AHEAD ? &gs.vals[which][((t8 * 2 + e) * NT + tid) * MT * 4]
                     : reinterpret_cast<const unsigned char*>(base + node * stride);
        const bool on = P::AHEAD || node < d.n;
        if constexpr (MT == 2) {
          uint2 u = make_uint2(0u, 0u);
          if (on) u = *reinterpret_cast<const uint2*>(src);
          r[t8][e][0] = u.x;
          r[t8][e][1] = u.y;
        } else {
          r[t8][e][0] = on ? *reinterpret_cast<const uint32_t*>(src) : 0u;
        }
      }
  };
  // B fragments of eight-row tiles r0 and r0 + 8, block kb: (k low, k high) of each
  const uint32_t kq0 = tc::smem_u32(&gs.kq[0][0]);
  const uint32_t b_lane = kq0 + (((lane >> 4) * 8 + (lane & 7)) * P::KP + ((lane >> 3) & 1) * 8) * 2;
  const auto frag2 = [&](int r0, int kb, uint32_t (&b)[4]) {
    mm::ldsm4(b, b_lane + (r0 * P::KP + kb * 16) * 2);
  };
  // gram tile -> first row, first column's row
  const auto tile_at = [&](int tile, int& row0, int& col0) {
    if constexpr (TN == 8) {
      row0 = 0;
      col0 = tile * 8;
    } else if (tile < 2 * TH) {
      const int half = tile / TH, rem = tile - half * TH;
      int mt = 0;
      while ((mt + 1) * (mt + 2) <= rem) ++mt;
      row0 = half * TN + mt * 16;
      col0 = (rem - mt * (mt + 1)) * 8;
    } else {
      row0 = TN + (tile - 2 * TH) / 2 * 16;
      col0 = TN + (tile - 2 * TH) * 8;
    }
    return tile < TILES;
  };
  float nwv[VC];
#pragma unroll
  for (int e = 0; e < VC; ++e) nwv[e] = NORM ? bf2f(a.nw[c + e]) : 1.f;

  int32_t* const flags = tid == 0 ? a.status : nullptr;
  DeltaRaw after = raw_nxt;
  DeltaUnit cur = unit_of(group, at_cur, raw_cur, flags);
  DeltaUnit nxt = unit_of(group + GROUPS, at_nxt, raw_nxt, flags);
  if (tid == 0) {
    fetch(group, cur);
    if constexpr (ST > GROUPS) fetch(group + GROUPS, nxt);
  }
  // three groups of copies are under way per thread and unit, in this order: rows,
  // values, gates; waiting for all but the last two is waiting for the next one
  load_rows(cur);
  copy_vals(0, a.v, a.vs, cur);
  tc::cp_async_commit();
  if constexpr (NORM) copy_vals(1, a.z, a.zs, cur);
  tc::cp_async_commit();
  const auto refill = [&](int i) {                   // unit i has used up its buffer
    if constexpr (ST == GROUPS) fetch(i + ST, nxt);
    else fetch(i + ST, unit_of(i + ST, at_nxt.step(ST - GROUPS, a.HV), raw_of(at_nxt.step(ST - GROUPS, a.HV)), nullptr));
  };
  int turn = 0;                                      // units computed: an empty one holds no warp up
  for (int i = group; i < count; i += GROUPS) {
    const DeltaAt at_after = at_nxt.step(GROUPS, a.HV);
    if (at_after.seq != at_nxt.seq) after = raw_of(at_after);
    const int n = cur.n;
    if (n == 0) {                                    // nothing to compute, and no copy: the buffer is free
      if (tid == 0) refill(i);
      tc::cp_async_wait<0>();                        // the next unit's rows go where these went
      load_rows(nxt);
      copy_vals(0, a.v, a.vs, nxt);
      tc::cp_async_commit();
      if constexpr (NORM) copy_vals(1, a.z, a.zs, nxt);
      tc::cp_async_commit();
    } else {
      int* par = gs.par[turn++ & 1];
      for (int j = tid; j < TN * (TN + 1); j += NT) (&gs.dec[0][0])[j] = 0.f;
      if (tid < TN) {
        const bool on = tid < n;
        par[tid] = on ? tree_parent(my_par, tid, a.status) : -1;
        gs.eg[tid] = on ? expf(my_g) : 0.f;
        gs.beta[tid] = on ? my_beta : 0.f;
      }
      tc::cp_async_wait<2>();
      group_sync();                                  // rows and scalars are there

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
      // gram tiles, the last warps first: the first ones walk the trees
      float gram[GT][4];
#pragma unroll
      for (int j = 0; j < GT; ++j) {
        int row0, col0;
#pragma unroll
        for (int e = 0; e < 4; ++e) gram[j][e] = 0.f;
        if (tile_at(NW - 1 - warp + j * NW, row0, col0)) {
          const uint32_t a_addr = kq0 + ((row0 + (lane & 15)) * P::KP + (lane >> 4) * 8) * 2;
          const uint32_t b_addr = kq0 + ((col0 + (lane & 7)) * P::KP + (lane >> 3) * 8) * 2;
#pragma unroll
          for (int kb = 0; kb < KB; kb += 2) {
            uint32_t f[4], b[4];
            mm::ldsm4(b, b_addr + kb * 32);
            mm::ldsm4(f, a_addr + kb * 32);
            mm::mma16816(gram[j], f, b[0], b[1]);
            mm::ldsm4(f, a_addr + kb * 32 + 32);
            mm::mma16816(gram[j], f, b[2], b[3]);
          }
          // the diagonal: norms
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = row0 + gr + (e >> 1) * 8;
            if (row == col0 + 2 * tq + (e & 1))
              gs.norm[row] = rsqrtf(gram[j][e] + 1e-6f) * (row < TN ? 1.f : a.scale);
          }
        }
      }

      // X^T = S_0^T [K; Q]^T
      await_state(i);
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
            for (int e = 0; e < 4; ++e) {
              const int j = (e >> 1) * 2, col = 2 * mt + (e & 1);
              mm::split2(s[j][col], s[j + 1][col], hi[mt][e], lo[mt][e]);
            }
#pragma unroll
          for (int t8 = 0; t8 < 2 * KT; t8 += 2) {
            uint32_t b[4];
            frag2(t8 * 8, kb, b);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                mm::mma16816(acc[t8 + u][mt], hi[mt], b[2 * u], b[2 * u + 1]);
                mm::mma16816(acc[t8 + u][mt], lo[mt], b[2 * u], b[2 * u + 1]);
              }
          }
        }
      }
      group_sync();                                  // decays complete; state and rows are used up
      if (gs.lost) break;                            // (set before this barrier only: all see the same)
      if (tid == 0) refill(i);
      load_rows(nxt);

      // gram tiles -> the factors -A and M
#pragma unroll
      for (int j = 0; j < GT; ++j) {
        int row0, col0;
        if (tile_at(NW - 1 - warp + j * NW, row0, col0) && col0 < TN) {
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
      tc::cp_async_wait<2>();
      uint32_t vr[KT][2][MT], zr[KT][2][MT];
      load_vals(vr, 0, a.v, a.vs, cur);
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
      copy_vals(0, a.v, a.vs, nxt);
      tc::cp_async_commit();
      group_sync();                                  // the factors are complete

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
            unsigned bad[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float4 t = make_float4(s[mt][0], s[mt][1], s[mt][2], s[mt][3]);
              bad[mt] = solve8_guarded<P::AP>(t, &gs.at[blk * 8][blk * 8], lane);
              r[mt][0] = t.x;
              r[mt][1] = t.y;
              r[mt][2] = t.z;
              r[mt][3] = t.w;
            }
            // (a sum in an accumulator that is NaN stays NaN)
#pragma unroll
            for (int t8 = blk; t8 < KT; ++t8)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const unsigned on = path_in_block(par, t8 * 8 + 2 * tq + e, blk);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  if (bad[mt] & on) acc[KT + t8][mt][e] = __int_as_float(0x7fffffff);
                  if (bad[mt] >> 8 & on) acc[KT + t8][mt][2 + e] = __int_as_float(0x7fffffff);
                }
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
        tc::cp_async_wait<2>();
        load_vals(zr, 1, a.z, a.zs, cur);
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
      if constexpr (NORM) copy_vals(1, a.z, a.zs, nxt);
      tc::cp_async_commit();
    }
    cur = nxt;
    nxt = unit_of(i + 2 * GROUPS, at_after, after, flags);
    at_nxt = at_after;
  }
  // a group that gave up leaves its units' outputs as they were; what it asked for may
  // still land in shared memory
  if (gs.lost) {
    tc::cp_async_wait<0>();
    if (tid == 0)
      for (int i = asked; i > asked - ST && i >= 0; i -= GROUPS)
        tc::mbar_wait(tc::smem_u32(&sm.full[i % ST]), (i / ST) & 1, kDeltaWait);
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
  GDN_UNSUPPORTED(units < (1ll << 30) && num_v_heads <= 65535, "%s: too many (sequence, head) units",
                  fn);
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
  const int rep = num_v_heads / num_k_heads;
  const DeltaArgs a{(const bf16*)q, (const bf16*)k, (const bf16*)v, q_row_stride, k_row_stride,
                    v_row_stride, g, (const bf16*)beta, num_slots, ids, cu_seqlens, parents,
                    max_nodes, n_tokens, (bf16*)out, num_v_heads, (int)units,
                    rep == 1 ? 0u : (unsigned)(((1ull << 32) + rep - 1) / rep), scale,
                    (const bf16*)z, z_row_stride, (const bf16*)norm_weight, norm_eps,
                    aligned16(q) && aligned16(k) && q_row_stride % 8 == 0 && k_row_stride % 8 == 0,
                    wait_limit(kDeltaWait), status};
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
