// Attention of drafted nodes over a paged cache: node i of sequence r sees the
// cache's positions [0, context_len) and, at context_len + j, the nodes j on its
// path (itself included), whose keys and values already stand in the cache.  One
// node per sequence is the plain decode step, a chain the causal one.
//
//   o_i = sum_p softmax_p(scale q_i.k_p) v_p
//
// HBM: every cached key and value of a sequence is read once (4 D bytes per
// position and kv-head), so the G = HQ / HKV query heads of a kv-head and all
// nodes form the rows of one tile of BM = 16 WM rows (more rows: further tiles).
//
// Work is cut evenly, whatever the sequences' lengths: all tiles of BN positions of
// all (sequence, kv-head, row tile) units in one line, of which each CTA takes an
// equal run; every CTA finds its place by a scan over the lengths.  A unit that one CTA
// holds whole is finished there; of one that is cut each CTA writes its rows' running
// maximum, sum and weighted values in fp32, and a second launch joins them.  (Chunks of
// a fixed length, one CTA each, left 128 sequences of 256 to 4352 positions at half the
// copy rate: half of the CTAs had nothing to do, the others started up for 10 tiles.)
//
// A producer warp brings the tiles by TMA (boxes of as many positions as divide a
// page, 128-byte swizzle) into a ring of stages, across unit borders; WM warps over
// rows x WN warps over positions run one pass with the softmax's running maximum
// and sum, scores and probabilities in registers (the score tile's accumulators are
// the next product's A operand).  Sums and statistics are fp32.  The second product takes
// the probabilities in bf16, as the values are: with 16 rows, where the traffic bounds it, as
// two parts (rounded, and what that leaves: 16 bits), which takes 0.7 % longer and leaves
// the output's own rounding as the only error of note (1.7e-3 relative to 64 bits); with
// more rows rounded once (2.1e-3 to 2.3e-3), as two parts take 11 to 19 % there with
// mma.sync (128 sequences of 8 nodes and 2303 positions 138 us instead of 123) and 8 % on
// tcgen05 (32 of 16 to 32 nodes 100 us instead of 92, the parts in TMEM).
//
// In the tiles that hold nodes or reach behind them, value rows behind the last node
// are zeroed in shared memory, and so are nodes' rows that are not finite, which must
// not reach nodes off their path (probability zero times NaN); the nodes that do see
// one of those get NaN outputs.  So does a whole sequence with a missing page, whose
// positions hold whatever tile stood in shared memory before.
#include "mma_util.cuh"
#include "tc_util.cuh"
#include "tmap.cuh"
#include "tree.cuh"

namespace gdn {

constexpr uint32_t kAttnWait = 1u << 22;      // polls
constexpr int kAttnSms = 148;

struct AttnArgs {
  const bf16* q;
  int64_t qs;
  int64_t num_blocks;
  int block_size, box;            // positions of a page, and of one TMA box (divides it)
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
  int HQ, HKV, G;
  int tile_rows;                  // rows of a row tile: BM, or on tcgen05 the whole nodes in it
  float scale_log2;
  int64_t* prefix;                // [n_seqs + 1]: tiles before each sequence's
  float* part_o;                  // [CTAs][2][D / 4][BM][4]: rows side by side
  float2* part_ml;                // [CTAs][2][BM]: maximum (base 2; NaN: no part, the CTA gave up), sum
  uint32_t wait;                  // polls
  int32_t* status;
};

// A wait that runs out (never, unless a copy is lost) ends the CTA's work: `lost` of the
// thread, flagged in the status word.  A thread that is lost waits for nothing more, issues
// no copy and no product, arrives at no barrier and clears no values; it runs through the
// rest of the CTA's tiles all the same, as the named barriers count it.  Threads that
// depend on it run out of polls in their turn, once each.  Rows that may hold anything of
// this are not written, and their parts say so to the joining kernel.
__device__ __forceinline__ void attn_wait(unsigned long long& bar, uint32_t parity, bool& lost,
                                          const AttnArgs& a) {
  if (lost || tc::mbar_wait(tc::smem_u32(&bar), parity, a.wait)) return;
  lost = true;
  if (a.status) atomicOr(a.status, GDN_STATUS_TIMEOUT);
}

// What was issued lands before the CTA ends (the normal limit, whatever a test has set).
__device__ __forceinline__ void attn_drain(unsigned long long& bar, uint32_t parity) {
  tc::mbar_wait(tc::smem_u32(&bar), parity, kAttnWait);
}

// A sequence as attention sees it; n = 0: nothing to compute.
struct AttnSeq {
  int64_t start;
  int n, ctx, tiles, row_tiles;
};

template <int BM, int BN>
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, int r, int32_t* status) {
  AttnSeq s{0, 0, 0, 0, 0};
  int n;
  if (!tree_rows(a.cu, r, a.n_tokens, a.max_nodes, status, s.start, n) || n == 0) return s;
  const int c = a.ctx[r];
  if (c < 0 || (int64_t)c + n > a.max_len) {
    if (status) atomicOr(status, GDN_STATUS_BAD_SEQLEN);
    return s;
  }
  s.n = n;
  s.ctx = c;
  s.tiles = (c + n + BN - 1) / BN;
  const int rows = BM == 128 ? a.tile_rows : BM;     // (a constant divides faster)
  s.row_tiles = (n * a.G + rows - 1) / rows;
  return s;
}

// Shared memory of the scan that finds a CTA's run of tiles.
struct AttnScan {
  int64_t base;
  int warp[12], seq;
};

// The CTA's run [w0, w1) of all units' tiles, the sequence it begins in and that one's
// first tile; false: none.  All threads (NW warps) take part; the sequences are scanned
// in strips of a thread each.  CTA 0 also leaves every sequence's first tile for the
// joining kernel, and flags malformed sequences.
template <int BM, int BN, int NW>
__device__ __forceinline__ bool attn_run(const AttnArgs& a, AttnScan& sc, int64_t& w0, int64_t& w1,
                                         int& seq, int64_t& seq_base) {
  constexpr int NT = 32 * NW;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const auto weight = [&](int r, int32_t* status) -> int64_t {
    if (r >= a.n_seqs) return 0;
    const AttnSeq s = attn_seq<BM, BN>(a, r, status);
    return (int64_t)s.tiles * s.row_tiles * a.HKV;
  };
  const auto strip_sum = [&](int64_t v) {            // the sum before this thread, and of all
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    // a strip's tiles fit 31 bits: at most 384 sequences of 2^22 tiles (host check)
    __syncthreads();
    if (lane == 31) sc.warp[warp] = (int)inc;
    __syncthreads();
    int64_t before = inc - v, all = 0;
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += sc.warp[w];
      all += sc.warp[w];
    }
    return make_longlong2(before, all);
  };
  int64_t total = 0;
  const bool scribe = blockIdx.x == 0;
  longlong2 first{0, 0};
  for (int s0 = 0; s0 < a.n_seqs; s0 += NT) {
    const longlong2 st = strip_sum(weight(s0 + tid, scribe ? a.status : nullptr));
    if (s0 == 0) first = st;
    if (scribe && s0 + tid < a.n_seqs) a.prefix[s0 + tid] = total + st.x;
    total += st.y;
  }
  if (scribe && tid == 0) a.prefix[a.n_seqs] = total;
  // no run is empty: fewer tiles than CTAs go to as many CTAs
  const int64_t ctas = min((int64_t)gridDim.x, total);
  if (blockIdx.x >= ctas) return false;
  w0 = total * blockIdx.x / ctas;
  w1 = total * (blockIdx.x + 1) / ctas;
  int64_t base = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += NT) {
    const int64_t v = weight(s0 + tid, nullptr);
    const longlong2 st = a.n_seqs <= NT ? first : strip_sum(v);
    const int64_t at = base + st.x;
    if (w0 >= at && w0 < at + v) {
      sc.seq = s0 + tid;
      sc.base = at;
    }
    base += st.y;
    if (base > w0) break;
  }
  __syncthreads();
  seq = sc.seq;
  seq_base = sc.base;
  return true;
}

// The producer warp's part of a segment: `seg` tiles from tile0 on into the ring of
// stages (tile number `it` of this CTA comes first).  A lane per box looks its page up,
// 32 boxes ahead; a missing page is flagged and not read, and `gone` of its stage and of
// the segment's later ones says so.
template <int D, int BN, int ST>
__device__ __forceinline__ void attn_produce(const AttnArgs& a, const CUtensorMap& kmap,
                                             const CUtensorMap& vmap, uint32_t kv0,
                                             unsigned long long* fulls, unsigned long long* empties,
                                             int* gone, int seq, int kvh, int len, int tile0, int seg, int it,
                                             bool& lost, int& issued) {
  constexpr int HALVES = D / 64;
  const int lane = threadIdx.x & 31;
  const int per_tile = BN / a.box;                   // boxes of a tile
  unsigned missed = 0;
  for (int b0 = 0; b0 < seg * per_tile; b0 += 32) {
    const int p_box = (tile0 * per_tile + b0 + lane) * a.box;
    int page = -2, row = 0;                          // -2: nothing to load
    bool bad = false;
    if (b0 + lane < seg * per_tile && p_box < len) {
      const int blk = p_box / a.block_size;
      row = p_box - blk * a.block_size;
      page = blk < a.max_blocks ? a.tables[seq * a.table_stride + blk] : -1;
      if (page < 0 || page >= a.num_blocks) {
        if (a.status) atomicOr(a.status, GDN_STATUS_BAD_SLOT);
        page = -2;
        bad = true;
      }
    }
    const unsigned there = __ballot_sync(0xffffffffu, page >= 0), lack = __ballot_sync(0xffffffffu, bad);
    const int boxes = min(32, seg * per_tile - b0);
    for (int i = 0; i < boxes; ++i) {
      const int in_tile = (b0 + i) % per_tile;
      const int t = it + (b0 + i) / per_tile, stage = t % ST;
      const int pg = __shfl_sync(0xffffffffu, page, i), rw = __shfl_sync(0xffffffffu, row, i);
      if (lane == 0) {
        const uint32_t full = tc::smem_u32(&fulls[stage]);
        if (in_tile == 0) {
          attn_wait(empties[stage], ((t / ST) & 1) ^ 1, lost, a);
          if (!lost) issued = t + 1;
        }
        if (!lost && (in_tile == 0 || i == 0)) {
          // the boxes of this tile that this round of 32 issues; the tile's last
          // round makes the arrival
          const int m = min(per_tile - in_tile, boxes - i);
          const unsigned of_tile = m == 32 ? 0xffffffffu : (1u << m) - 1;
          const uint32_t bytes = (uint32_t)__popc(there >> i & of_tile) * a.box * D * 4;
          missed |= lack >> i & of_tile;
          if (in_tile + m == per_tile) {
            gone[stage] = missed != 0;
            tc::mbar_expect_tx(full, bytes);
          } else {
            asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(full), "r"(bytes)
                         : "memory");
          }
        }
        if (!lost && pg >= 0) {
#pragma unroll
          for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int hf = 0; hf < HALVES; ++hf)
              asm volatile(
                  "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
                  "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                      kv0 + ((stage * 2 + kv) * HALVES + hf) * (BN * 128) + in_tile * a.box * 128),
                  "l"(kv == 0 ? &kmap : &vmap), "r"(hf * 64), "r"(kvh), "r"(rw), "r"(pg), "r"(full)
                  : "memory");
        }
      }
      __syncwarp();
    }
  }
  lost = __shfl_sync(0xffffffffu, lost, 0);
}

// The producer warp's last tiles have landed.
template <int ST>
__device__ __forceinline__ void attn_produced(unsigned long long* fulls, int issued) {
  if ((threadIdx.x & 31) == 0)
    for (int t = max(0, issued - ST); t < issued; ++t) attn_drain(fulls[t % ST], (t / ST) & 1);
}

template <int D, int WM, int WN>
struct Attn {
  static constexpr int BM = 16 * WM, NC = WM * WN;               // NC: consumer warps
  static constexpr int BN = D == 64 ? 128 : 64;                   // positions of a tile: 32 KB and more
  static constexpr int WT = BN / WN;                              // positions per warp
  static constexpr int HALVES = D / 64;                           // 128-byte column blocks
  static constexpr int CTAS = D <= 128 ? 2 : 1;                   // per SM
  static constexpr int STAGE = 2 * BN * D * 2;                    // bytes of keys and values
  static constexpr int ST = 3;
  static constexpr int PARTS = WM == 1 ? 2 : 1;                   // of a probability
  struct Smem {
    __align__(1024) unsigned char kv[ST][2][HALVES][BN * 128];
    __align__(16) float join[WN > 1 ? WN * BM * 36 : 4];          // 32 columns at a time
    float2 ml[WN > 1 ? WN * BM : 1];
    unsigned long long anc[kMaxTreeNodes];
    unsigned long long full[ST], empty[ST], bad;
    AttnScan scan;
    int par[kMaxTreeNodes], gone[ST], lost, issued;
  };
};

// 2^x by the hardware's instruction (2 ulp; results below 2^-126 become zero).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Byte offset of 16-byte piece c of row r in a [HALVES][BN] tile of 128-byte swizzled rows.
template <int BN>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  return (uint32_t)((c >> 3) * (BN * 128) + r * 128 + (((c ^ r) & 7) << 4));
}

template <int D, int WM, int WN>
__global__ void __launch_bounds__(32 * (WM * WN + 1), Attn<D, WM, WN>::CTAS)
    attention_tree_kernel(const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, const AttnArgs a) {
  using P = Attn<D, WM, WN>;
  constexpr int NC = P::NC, BM = P::BM, BN = P::BN, WT = P::WT, ST = P::ST;
  static_assert(WT % 16 == 0, "a warp takes whole 16-position blocks");
  extern __shared__ unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<typename P::Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      tc::mbar_init(tc::smem_u32(&sm.full[i]), 1);
      tc::mbar_init(tc::smem_u32(&sm.empty[i]), NC);
    }
    tc::mbar_init_fence();
    sm.lost = sm.issued = 0;
  }
  int64_t w0, w1, seq_base;
  int seq;
  if (!attn_run<BM, BN, NC + 1>(a, sm.scan, w0, w1, seq, seq_base)) return;

  // ---- the run, a segment (part of a unit) at a time; every warp keeps the same place ----
  int it = 0;                                        // tiles of this CTA so far
  bool lost = false;
  AttnSeq s = attn_seq<BM, BN>(a, seq, nullptr);
  for (int64_t w = w0; w < w1;) {
    const int mine = s.tiles * s.row_tiles * a.HKV;  // at most 2^22 (host check)
    if (w >= seq_base + mine) {
      seq_base += mine;
      s = attn_seq<BM, BN>(a, ++seq, nullptr);
      continue;
    }
    const int local = (int)(w - seq_base), unit = local / s.tiles, tile0 = local - unit * s.tiles;
    const int kvh = unit / s.row_tiles, rt = unit - kvh * s.row_tiles;
    const int seg = (int)min((int64_t)(s.tiles - tile0), w1 - w);
    const int len = s.ctx + s.n;

    if (warp == NC) {
      if (!lost)
        attn_produce<D, BN, ST>(a, kmap, vmap, tc::smem_u32(&sm.kv[0][0][0][0]), sm.full, sm.empty, sm.gone,
                                seq, kvh, len, tile0, seg, it, lost, sm.issued);
    } else {
      // ---- consumers ----
      const auto sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(NC * 32) : "memory"); };
      const int gr = lane >> 2, tq = lane & 3, wm = warp / WN, wn = warp - wm * WN;
      const int row0 = rt * BM, rows = s.n * a.G;    // rows: node * G + head within the group
      const int my_row[2] = {row0 + wm * 16 + gr, row0 + wm * 16 + gr + 8};
      const bool idle = row0 + wm * 16 >= rows;      // no row of this warp exists
      const bool masks = (tile0 + seg) * BN > s.ctx; // the segment reaches the nodes
      if (masks) {
        if (tid < s.n) sm.par[tid] = tree_parent(a.parents[s.start + tid], tid, a.status);
        if (tid == 0) sm.bad = 0;
        sync();
        if (tid < s.n) {
          unsigned long long m = 0;
          for (int j = tid; j >= 0; j = sm.par[j]) m |= 1ull << j;
          sm.anc[tid] = m;
        }
      }
      int node[2];
      const bf16* qp[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        node[hh] = min(my_row[hh], rows - 1) / a.G;
        qp[hh] = a.q + (s.start + node[hh]) * a.qs +
                 (int64_t)(kvh * a.G + min(my_row[hh], rows - 1) - node[hh] * a.G) * D + 2 * tq;
      }
      uint32_t qa[D / 16][4];
#pragma unroll
      for (int kb = 0; kb < D / 16; ++kb) {
        qa[kb][0] = *reinterpret_cast<const uint32_t*>(qp[0] + kb * 16);
        qa[kb][1] = *reinterpret_cast<const uint32_t*>(qp[1] + kb * 16);
        qa[kb][2] = *reinterpret_cast<const uint32_t*>(qp[0] + kb * 16 + 8);
        qa[kb][3] = *reinterpret_cast<const uint32_t*>(qp[1] + kb * 16 + 8);
      }
      if (masks) sync();
      unsigned long long anc[2] = {0, 0};
      if (masks) {
        anc[0] = my_row[0] < rows ? sm.anc[node[0]] : 0ull;
        anc[1] = my_row[1] < rows ? sm.anc[node[1]] : 0ull;
      }

      float o[D / 8][4];
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

      for (int t = 0; t < seg; ++t) {
        const int stage = (it + t) % ST;
        attn_wait(sm.full[stage], ((it + t) / ST) & 1, lost, a);
        if (lost) sm.lost = 1;
        __syncwarp();
        if (t == seg - 1 && sm.gone[stage]) sum[0] = sum[1] = __int_as_float(0x7fffffff);   // and so the outputs
        const int p_tile = (tile0 + t) * BN;
        const bool edge = p_tile + BN > s.ctx;       // holds nodes or positions behind them
        if (edge) {
          unsigned char* vt = &sm.kv[stage][1][0][0];
          for (int i = tid; i < BN * (D / 8); i += NC * 32) {
            const int r = i / (D / 8), c = i - r * (D / 8), j = p_tile + r - s.ctx;
            if (j < 0 || lost) continue;
            uint4* p = reinterpret_cast<uint4*>(vt + tile_at<BN>(r, c));
            float f[8];
            unpack8(*p, f);
            bool finite = true;
#pragma unroll
            for (int e = 0; e < 8; ++e) finite &= fabsf(f[e]) <= 3.4e38f;
            if (j >= s.n || !finite) {
              *p = make_uint4(0, 0, 0, 0);
              if (j < s.n) atomicOr(&sm.bad, 1ull << j);
            }
          }
          sync();
        }
        if (!idle) {
          const uint32_t k_base = tc::smem_u32(&sm.kv[stage][0][0][0]);
          const uint32_t v_base = tc::smem_u32(&sm.kv[stage][1][0][0]);
          // XT positions at a time: their scores and probabilities stay in registers
          constexpr int XT = WT > 32 ? 32 : WT;
#pragma unroll
          for (int x0 = 0; x0 < WT; x0 += XT) {
            const int p0 = wn * WT + x0;               // first position within the tile
            float x[XT / 8][4];
#pragma unroll
            for (int i = 0; i < XT / 8; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
#pragma unroll
            for (int kb = 0; kb < D / 16; ++kb)
#pragma unroll
              for (int i = 0; i < XT / 8; i += 2) {
                uint32_t b[4];
                mm::ldsm4(b, k_base + tile_at<BN>(p0 + i * 8 + (lane >> 4) * 8 + (lane & 7),
                                                  kb * 2 + ((lane >> 3) & 1)));
                mm::mma16816(x[i], qa[kb], b[0], b[1]);
                mm::mma16816(x[i + 1], qa[kb], b[2], b[3]);
              }
            if (edge) {
#pragma unroll
              for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int i = 0; i < XT / 8; ++i)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const int j = p_tile + p0 + i * 8 + 2 * tq + e - s.ctx;
                    const bool seen = j < 0 || (j < s.n && (anc[hh] >> (j & 63) & 1));
                    if (!seen) x[i][hh * 2 + e] = -INFINITY;
                  }
            }
            // running maximum and sum; scaled to base 2 (scale > 0) within the exponent's argument
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              float m = -INFINITY;
#pragma unroll
              for (int i = 0; i < XT / 8; ++i) m = fmaxf(m, fmaxf(x[i][hh * 2], x[i][hh * 2 + 1]));
              m *= a.scale_log2;
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
              m = fmaxf(m, mx[hh]);
              const float off = m == -INFINITY ? 0.f : m;    // a row that has seen nothing yet
              const float corr = ex2(mx[hh] - off);
              float add = 0.f;
#pragma unroll
              for (int i = 0; i < XT / 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float& v = x[i][hh * 2 + e];
                  v = ex2(fmaf(v, a.scale_log2, -off));
                  add += v;
                }
              sum[hh] = sum[hh] * corr + add;
              if (__any_sync(0xffffffffu, m != mx[hh])) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                  o[i][hh * 2] *= corr;
                  o[i][hh * 2 + 1] *= corr;
                }
              }
              mx[hh] = m;
            }
#pragma unroll
            for (int i = 0; i < XT / 16; ++i) {
              uint32_t pa[P::PARTS][4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float* f = &x[2 * i + (e >> 1)][(e & 1) * 2];
                if constexpr (P::PARTS == 2) mm::split2(f[0], f[1], pa[0][e], pa[1][e]);
                else pa[0][e] = mm::pack2(f[0], f[1]);
              }
#pragma unroll
              for (int c = 0; c < D / 8; c += 2) {
                uint32_t b[4];
                mm::ldsm4t(b, v_base + tile_at<BN>(p0 + i * 16 + (lane & 15), c + (lane >> 4)));
#pragma unroll
                for (int v = 0; v < P::PARTS; ++v) {
                  mm::mma16816(o[c], pa[v], b[0], b[1]);
                  mm::mma16816(o[c + 1], pa[v], b[2], b[3]);
                }
              }
            }
          }
        }
        if (edge) tc::fence_async_smem();            // our writes before the next copy's
        __syncwarp();
        if (lane == 0 && !lost) tc::mbar_arrive(tc::smem_u32(&sm.empty[stage]));
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        sum[hh] += __shfl_xor_sync(0xffffffffu, sum[hh], 1);
        sum[hh] += __shfl_xor_sync(0xffffffffu, sum[hh], 2);
      }
      const bool whole = tile0 == 0 && seg == s.tiles;
      const int64_t part = ((int64_t)blockIdx.x * 2 + (w == w0 ? 0 : 1)) * BM;
      const unsigned long long bad = masks ? *reinterpret_cast<volatile unsigned long long*>(&sm.bad) : 0;

      // a warp is lost with any of its lanes, and with a warp that was to clear values for it
      const float2 no_part = make_float2(__int_as_float(0x7fffffff), 0.f);

      if constexpr (WN == 1) {
        const bool failed = __any_sync(0xffffffffu, lost || *reinterpret_cast<volatile int*>(&sm.lost));
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          if (my_row[hh] >= rows) continue;
          const bool nan = (anc[hh] & bad) != 0;
          const float inv = whole ? 1.f / sum[hh] : 1.f;
          const int r = wm * 16 + gr + hh * 8;
          const int64_t at = (s.start + node[hh]) * a.HQ + kvh * a.G + my_row[hh] - node[hh] * a.G;
          if (!whole && tq == 0) a.part_ml[part + r] = failed ? no_part : make_float2(mx[hh], sum[hh]);
          if (failed) continue;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            float u = o[i][hh * 2] * inv, v = o[i][hh * 2 + 1] * inv;
            if (nan) u = v = __int_as_float(0x7fffffff);
            if (whole)
              *reinterpret_cast<uint32_t*>(a.out + at * D + i * 8 + 2 * tq) = mm::pack2(u, v);
            else
              *reinterpret_cast<float2*>(a.part_o + part * D +
                                         ((i * 2 + (tq >> 1)) * BM + r) * 4 + (tq & 1) * 2) =
                  make_float2(u, v);
          }
        }
        if (masks) sync();                           // the masks are used up
      } else {
        // join the WN warps of a row tile: common maximum, then 32 columns at a time
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
          if (tq == 0) sm.ml[wn * BM + wm * 16 + gr + hh * 8] = make_float2(mx[hh], sum[hh]);
        sync();
        // (no consumer waits for a tile between this barrier and the next: all see the same)
        const bool failed = *reinterpret_cast<volatile int*>(&sm.lost) != 0;
        float inv[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int r = wm * 16 + gr + hh * 8;
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int v = 0; v < WN; ++v) m = fmaxf(m, sm.ml[v * BM + r].x);
          const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int v = 0; v < WN; ++v) {
            const float2 p = sm.ml[v * BM + r];
            l = fmaf(p.y, ex2(p.x - off), l);
          }
          inv[hh] = ex2(mx[hh] - off) * (whole ? 1.f / l : 1.f);
          if (anc[hh] & bad) inv[hh] = __int_as_float(0x7fffffff);
          if (!whole && wn == 0 && tq == 0 && my_row[hh] < rows)
            a.part_ml[part + r] = failed ? no_part : make_float2(m, l);
        }
#pragma unroll
        for (int cq = 0; cq < D / 32; ++cq) {
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float2*>(
                  &sm.join[(wn * BM + wm * 16 + gr + hh * 8) * 36 + i * 8 + 2 * tq]) =
                  make_float2(o[cq * 4 + i][hh * 2] * inv[hh], o[cq * 4 + i][hh * 2 + 1] * inv[hh]);
          sync();
          for (int i = tid; i < BM * 8; i += NC * 32) {
            // a whole unit's rows are written along their columns, parts along the rows
            const int r = whole ? i >> 3 : i % BM, c = (whole ? i & 7 : i / BM) * 4, row = row0 + r;
            if (row < rows && !failed) {
              float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int v = 0; v < WN; ++v) {
                const float4 u = *reinterpret_cast<const float4*>(&sm.join[(v * BM + r) * 36 + c]);
                acc.x += u.x;
                acc.y += u.y;
                acc.z += u.z;
                acc.w += u.w;
              }
              if (whole) {
                const int nd = row / a.G;
                const int64_t at = (s.start + nd) * a.HQ + kvh * a.G + row - nd * a.G;
                *reinterpret_cast<uint2*>(a.out + at * D + cq * 32 + c) =
                    make_uint2(mm::pack2(acc.x, acc.y), mm::pack2(acc.z, acc.w));
              } else {
                *reinterpret_cast<float4*>(a.part_o + part * D + ((cq * 32 + c) / 4 * BM + r) * 4) = acc;
              }
            }
          }
          sync();
        }
      }
    }
    it += seg;
    w += seg;
  }
  if (warp == NC) attn_produced<ST>(sm.full, sm.issued);
}

// ---------------------------------------------------------------------------
// Many rows (more than 32 of a unit): the same on tcgen05, 128 rows to a tile.
//
// mma.sync reaches a quarter of the tensor cores' rate, and 128 rows need 64 products
// per byte: with it, 32 trees of 16 to 32 nodes over 4 to 8 thousand positions took
// 214 us against 62 of memory traffic.  Here S = Q K^T (128 x 64) and O += P V (128 x D)
// are issued by a thread each, from shared memory into TMEM; two groups of four warps, a
// thread per row, take the tiles in turn: read S (no exchange between lanes), write P as
// bf16 into shared memory and correct O.  Each group has its own S, P, running maximum, sum
// and O, joined at the end of a segment, so that the two chains of a tile (product,
// softmax, product) never wait for one another (one group and one issuing thread: 144
// us).  The TMA producer keeps ST - 1 further tiles under way, and one more warp brings the
// next segment's queries (a box of whole nodes' heads) and its nodes' ancestors: what a
// segment does once is what is left above the memory traffic (queries through registers
// when the segment began: 105 us, now 92; a longer context costs 6.3 TB/s).
//
// O is corrected only when a row's maximum has grown by more than 2^8 since its last
// correction: until then its probabilities are measured against the older maximum, which
// the final division cancels.
// ---------------------------------------------------------------------------
template <int D>
struct AttnTc {
  static constexpr int BM = 128, BN = 64, HALVES = D / 64, ST = D == 64 ? 8 : 4;
  static constexpr uint32_t kColS = 0, kColO = 128, kCols = D == 64 ? 256 : 512;   // two of each
  struct Smem {
    __align__(1024) unsigned char kv[ST][2][HALVES][BN * 128];
    __align__(1024) unsigned char q[2][HALVES][BM * 128];           // of two segments, as anc and bad
    __align__(1024) unsigned char p[2][BM * 128];
    unsigned long long anc[2][kMaxTreeNodes], bad[2];
    unsigned long long full[ST], empty[ST], s_full[2], s_free[2], p_full[2], pv_done[2], q_full[2],
        q_empty[2], anc_full[2];
    AttnScan scan;
    uint32_t tmem;
    int par[kMaxTreeNodes], gone[ST], lost;
  };
};

template <int D>
__global__ void __launch_bounds__(384, 1)
    attention_tree_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                             const __grid_constant__ CUtensorMap vmap,
                             const __grid_constant__ CUtensorMap qmap, const AttnArgs a) {
  using P = AttnTc<D>;
  constexpr int BM = P::BM, BN = P::BN, ST = P::ST;
  extern __shared__ unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<typename P::Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const auto bar = [](unsigned long long& b) { return tc::smem_u32(&b); };

  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      tc::mbar_init(bar(sm.full[i]), 1);
      tc::mbar_init(bar(sm.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(bar(sm.s_full[i]), 1);
      tc::mbar_init(bar(sm.s_free[i]), 4);
      tc::mbar_init(bar(sm.p_full[i]), 4);
      tc::mbar_init(bar(sm.pv_done[i]), 1);
      tc::mbar_init(bar(sm.q_full[i]), 1);
      tc::mbar_init(bar(sm.anc_full[i]), 1);
      tc::mbar_init(bar(sm.q_empty[i]), 9);           // the last S, and the softmax warps
    }
    tc::mbar_init_fence();
    sm.lost = 0;                                     // set by softmax threads alone
  }
  int64_t w0, w1, seq_base;
  int seq;
  if (!attn_run<BM, BN, 12>(a, sm.scan, w0, w1, seq, seq_base)) return;
  if (warp == 9) tc::tmem_alloc(tc::smem_u32(&sm.tmem), P::kCols);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = sm.tmem;

  bool lost = false;
  const auto wait = [&](unsigned long long& b, uint32_t parity) { attn_wait(b, parity, lost, a); };

  int it = 0, segs = 0;                              // tiles and segments of this CTA so far
  int issued = 0;                                    // what the warp's lane 0 has under way goes up to here
  AttnSeq s = attn_seq<BM, BN>(a, seq, nullptr);
  for (int64_t w = w0; w < w1;) {
    const int mine = s.tiles * s.row_tiles * a.HKV;  // at most 2^22 (host check)
    if (w >= seq_base + mine) {
      seq_base += mine;
      s = attn_seq<BM, BN>(a, ++seq, nullptr);
      continue;
    }
    const int local = (int)(w - seq_base), unit = local / s.tiles, tile0 = local - unit * s.tiles;
    const int kvh = unit / s.row_tiles, rt = unit - kvh * s.row_tiles;
    const int seg = (int)min((int64_t)(s.tiles - tile0), w1 - w);

    if (warp == 8) {
      if (!lost)
        attn_produce<D, BN, ST>(a, kmap, vmap, tc::smem_u32(&sm.kv[0][0][0][0]), sm.full, sm.empty, sm.gone,
                                seq, kvh, s.ctx + s.n, tile0, seg, it, lost, issued);
    } else if (warp == 11) {
      // ---- the segment's queries and ancestors, while the one before is worked on ----
      const int b = segs & 1;
      wait(sm.q_empty[b], ((segs >> 1) & 1) ^ 1);
      lost = __any_sync(0xffffffffu, lost);
      if (lane == 0 && !lost) {
        issued = segs + 1;
        tc::mbar_expect_tx(bar(sm.q_full[b]), (uint32_t)a.tile_rows * D * 2);
#pragma unroll
        for (int hf = 0; hf < P::HALVES; ++hf)
          tc::tma_load_3d(tc::smem_u32(&sm.q[b][hf][0]), &qmap, hf * 64, kvh * a.G,
                          (int)s.start + rt * (a.tile_rows / a.G), bar(sm.q_full[b]));
      }
      if ((tile0 + seg) * BN > s.ctx && !lost) {     // the segment reaches the nodes
        for (int j = lane; j < s.n; j += 32) sm.par[j] = tree_parent(a.parents[s.start + j], j, a.status);
        __syncwarp();
        for (int j = lane; j < s.n; j += 32) {
          unsigned long long m = 0;
          for (int x = j; x >= 0; x = sm.par[x]) m |= 1ull << x;
          sm.anc[b][j] = m;
        }
        if (lane == 0) sm.bad[b] = 0;
        __syncwarp();
      }
      if (lane == 0 && !lost) tc::mbar_arrive(bar(sm.anc_full[b]));
      __syncwarp();
    } else if (warp >= 9) {
      // ---- products: a thread for S, one for O.  (One thread for both took 2200 cycles
      // a tile, most of them instructions; hence also descriptors made once, of which a
      // step advances the address field.) ----
      if (lane == 0 && warp == 9) {
        wait(sm.q_full[segs & 1], (segs >> 1) & 1);
        const uint64_t qd = tc::smem_desc(tc::smem_u32(&sm.q[segs & 1][0][0]), 16, 1024);
        for (int T = it; T < it + seg; ++T) {
          wait(sm.full[T % ST], (T / ST) & 1);
          wait(sm.s_free[T & 1], ((T >> 1) & 1) ^ 1);
          if (lost) break;
          tc::fence_after();
          const uint64_t kd = tc::smem_desc(tc::smem_u32(&sm.kv[T % ST][0][0][0]), 16, 1024);
#pragma unroll
          for (int x = 0; x < D / 16; ++x)
            tc::mma_bf16(tmem + P::kColS + (T & 1) * 64,
                         qd + ((x >> 2) * (BM * 128) + (x & 3) * 32) / 16,
                         kd + ((x >> 2) * (BN * 128) + (x & 3) * 32) / 16,
                         tc::idesc_bf16(BM, BN, false, false), x > 0);
          tc::mma_commit(bar(sm.s_full[T & 1]));
          issued = T + 1;
        }
        if (!lost) tc::mma_commit(bar(sm.q_empty[segs & 1]));
      } else if (lane == 0) {
        for (int t = 0; t < seg; ++t) {
          const int T = it + t;
          wait(sm.full[T % ST], (T / ST) & 1);
          wait(sm.p_full[T & 1], (T >> 1) & 1);
          if (lost) break;
          tc::fence_after();
          const uint64_t pd = tc::smem_desc(tc::smem_u32(&sm.p[T & 1][0]), 16, 1024);
          const uint64_t vd = tc::smem_desc(tc::smem_u32(&sm.kv[T % ST][1][0][0]), BN * 128, 1024);
#pragma unroll
          for (int x = 0; x < BN / 16; ++x)
            tc::mma_bf16(tmem + P::kColO + (T & 1) * D, pd + x * 32 / 16, vd + x * 2048 / 16,
                         tc::idesc_bf16(BM, D, false, true), (t > 1 || x > 0) ? 1u : 0u);
          tc::mma_commit(bar(sm.empty[T % ST]));
          tc::mma_commit(bar(sm.pv_done[T & 1]));
          issued = T + 1;
        }
      }
      __syncwarp();
    } else {
      // ---- softmax: a thread per row and group; group g takes the tiles of parity g ----
      const auto sync_all = [&]() { asm volatile("bar.sync 3, 256;" ::: "memory"); };
      const int grp = warp >> 2, r = tid & 127;
      const int row = rt * a.tile_rows + r;
      const int rows = r < a.tile_rows ? s.n * a.G : 0;      // 0: no row of this thread's
      const int node = row < rows ? row / a.G : 0;
      const int64_t at = (s.start + node) * a.HQ + kvh * a.G + row - node * a.G;
      const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);

      float ref = -INFINITY, sum = 0.f;              // base 2: what the probabilities are measured against
      for (int t = (grp ^ it) & 1; t < seg; t += 2) {
        const int T = it + t, p_tile = (tile0 + t) * BN;
        const bool edge = p_tile + BN > s.ctx;       // holds nodes or positions behind them
        unsigned long long anc = 0;
        if (edge || t + 2 >= seg) wait(sm.full[T % ST], (T / ST) & 1);
        if (t + 2 >= seg && sm.gone[T % ST]) sum = __int_as_float(0x7fffffff);   // and so the outputs
        if (edge) {
          wait(sm.anc_full[segs & 1], (segs >> 1) & 1);
          if (row < rows) anc = sm.anc[segs & 1][node];
          unsigned char* vt = &sm.kv[T % ST][1][0][0];
#pragma unroll 4
          for (int i = r; i < BN * (D / 8); i += 128) {
            const int vrow = i / (D / 8), c = i - vrow * (D / 8), j = p_tile + vrow - s.ctx;
            if (j < 0 || lost) continue;
            uint4* p = reinterpret_cast<uint4*>(vt + tile_at<BN>(vrow, c));
            float f[8];
            unpack8(*p, f);
            bool finite = true;
#pragma unroll
            for (int e = 0; e < 8; ++e) finite &= fabsf(f[e]) <= 3.4e38f;
            if (j >= s.n || !finite) {
              *p = make_uint4(0, 0, 0, 0);
              if (j < s.n) atomicOr(&sm.bad[segs & 1], 1ull << j);
            }
          }
        }
        wait(sm.s_full[grp], (T >> 1) & 1);
        __syncwarp();
        tc::fence_after();
        float x[2][32];
        tc::tmem_ld32x2(tl + P::kColS + grp * 64, tl + P::kColS + grp * 64 + 32, x[0], x[1]);
        tc::fence_before();
        __syncwarp();
        if (lane == 0 && !lost) tc::mbar_arrive(bar(sm.s_free[grp]));
        if (edge) {                                  // a bit per position that the row sees
          const int nodes_at = s.ctx - p_tile;       // > -64, as the tile holds a node
          const unsigned long long see =
              nodes_at >= 0 ? ((1ull << nodes_at) - 1) | anc << nodes_at : anc >> -nodes_at;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t bits = (uint32_t)(see >> 32 * h);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[h][i] = bits >> i & 1 ? x[h][i] : -INFINITY;
          }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; ++i) m4[i & 3] = fmaxf(m4[i & 3], x[i >> 5][i & 31]);
        const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2;
        const bool grown = m > ref + 8.f;            // (from -inf: the row's first positions)
        const float was = ref;
        if (grown) ref = m;
        const float off = ref == -INFINITY ? 0.f : ref;
        const float corr = grown ? ex2(was - off) : 1.f;
        float a4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          float& v = x[i >> 5][i & 31];
          v = ex2(fmaf(v, a.scale_log2, -off));
          a4[i & 3] += v;
        }
        sum = sum * corr + ((a4[0] + a4[1]) + (a4[2] + a4[3]));
        // the group's last product has read P and left O alone
        wait(sm.pv_done[grp], ((T >> 1) & 1) ^ 1);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(&sm.p[grp][tc::sw128(r, c * 8)]) = pack8(&x[c >> 2][(c & 3) * 8]);
        if (t > 1 && __any_sync(0xffffffffu, grown)) {
          tc::fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            float o[32];
            tc::tmem_ld32(tl + P::kColO + grp * D + c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= corr;
            tc::tmem_st32(tl + P::kColO + grp * D + c, o);
          }
          tc::tmem_wait_st();
        }
        tc::fence_async_smem();                      // P and the zeroed values, before the product reads them
        tc::fence_before();
        if (edge) asm volatile("bar.sync %0, 128;" ::"r"(grp + 1) : "memory");   // every value row is clean
        else __syncwarp();
        if (lane == 0 && !lost) tc::mbar_arrive(bar(sm.p_full[grp]));
      }
      // join the groups: each waits for its own last product, which leaves its P free
      bool has[2];
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int T = it + seg - 1 - ((it + seg - 1 - v) & 1);   // the last tile of parity v
        has[v] = T >= it;
        if (has[v] && v == grp) wait(sm.pv_done[v], (T >> 1) & 1);
      }
      const bool masks = (tile0 + seg) * BN > s.ctx;
      if (masks) wait(sm.anc_full[segs & 1], (segs >> 1) & 1);
      if (lost) sm.lost = 1;
      __syncwarp();
      const auto ml = [&](int g) -> float2& { return reinterpret_cast<float2*>(&sm.p[g][0])[r]; };
      ml(grp) = make_float2(ref, sum);
      tc::fence_before();
      sync_all();
      tc::fence_after();
      // (no thread that sets it waits between this barrier and the next: all see the same)
      const bool failed = *reinterpret_cast<volatile int*>(&sm.lost) != 0;
      const float2 ml0 = ml(0), ml1 = ml(1);
      const float top = fmaxf(ml0.x, ml1.x), off = top == -INFINITY ? 0.f : top;
      float f0 = ex2(ml0.x - off), f1 = ex2(ml1.x - off);
      const float l = ml0.y * f0 + ml1.y * f1;
      const bool whole = tile0 == 0 && seg == s.tiles;
      const int64_t part = ((int64_t)blockIdx.x * 2 + (w == w0 ? 0 : 1)) * BM;
      bool nan = false;                              // the row sees a value row that is not finite
      if (masks)
        nan = row < rows && (sm.anc[segs & 1][node] &
                             *reinterpret_cast<volatile unsigned long long*>(&sm.bad[segs & 1])) != 0;
      const float inv = nan ? __int_as_float(0x7fffffff) : whole ? 1.f / l : 1.f;
      f0 *= inv;
      f1 *= inv;
      if (!whole && grp == 0 && row < rows)
        a.part_ml[part + r] = failed ? make_float2(__int_as_float(0x7fffffff), 0.f) : make_float2(top, l);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int c = grp * (D / 2) + i * 32;        // a half of the columns each
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.f;
#pragma unroll
        for (int v = 0; v < 2; ++v)
          if (has[v]) {
            float y[32];
            tc::tmem_ld32(tl + P::kColO + v * D + c, y);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(y[e], v == 0 ? f0 : f1, o[e]);
          }
        if (row < rows && !failed) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(a.out + at * D + c + e) = pack8(o + e);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(a.part_o + part * D + ((c + e) / 4 * BM + r) * 4) =
                  make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
      }
      tc::fence_before();
      sync_all();                                    // masks and O are used up
      if (lane == 0 && !lost) tc::mbar_arrive(bar(sm.q_empty[segs & 1]));
    }
    it += seg;
    ++segs;
    w += seg;
  }
  // what is under way ends before the CTA does, and before its TMEM is given back
  if (warp == 8) attn_produced<ST>(sm.full, issued);
  if (lane == 0 && issued > 0) {
    if (warp == 9) attn_drain(sm.s_full[(issued - 1) & 1], ((issued - 1) >> 1) & 1);
    if (warp == 10) attn_drain(sm.pv_done[(issued - 1) & 1], ((issued - 1) >> 1) & 1);
    if (warp == 11)
      for (int i = max(0, issued - 2); i < issued; ++i) attn_drain(sm.q_full[i & 1], (i >> 1) & 1);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 9) tc::tmem_dealloc(tmem, P::kCols);
}

// Joins the parts of a unit that was cut: a thread per row and 16 columns, threads side
// by side on rows.  SHARES of them split a row's parts, 8 where there are far fewer units
// than CTAs and hence many parts to each.  (A warp per row took 11 us instead of 7 for
// 32 sequences of 6144 positions and 32 nodes; launched early, to wait on the device for
// the first kernel's end, the two took 2 us longer.)
template <int D, int BM, int SHARES>
struct AttnJoin {
  static constexpr int RT = BM < 128 / SHARES ? BM : 128 / SHARES;   // rows per CTA
  static constexpr int CG = 128 / SHARES / RT < D / 16 ? 128 / SHARES / RT : D / 16;   // column groups
  static constexpr int kThreads = SHARES * RT * CG;
  static constexpr int kBlocksY = BM / RT * (D / 16 / CG);
  static_assert(D / 16 % CG == 0 && BM % RT == 0, "whole blocks");
};

template <int D, int BM, int BN, int SHARES>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttnArgs a, int max_row_tiles,
                                                             int grid) {
  using J = AttnJoin<D, BM, SHARES>;
  __shared__ float s_o[SHARES > 1 ? SHARES : 1][SHARES > 1 ? 17 * J::RT : 1];
  __shared__ float2 s_ml[SHARES][J::RT];
  const int per_seq = a.HKV * max_row_tiles;
  const int seq = blockIdx.x / per_seq, u = blockIdx.x - seq * per_seq;
  const int64_t base = a.prefix[seq], total = a.prefix[a.n_seqs];
  const AttnSeq s = attn_seq<BM, BN>(a, seq, nullptr);
  if (s.n == 0 || u >= a.HKV * s.row_tiles) return;
  const int64_t ctas = min((int64_t)grid, total);
  const int64_t u0 = base + (int64_t)u * s.tiles, u1 = u0 + s.tiles;
  // the CTA that holds tile w: the last b with total * b / ctas <= w
  const int b0 = (int)(((u0 + 1) * ctas - 1) / total), b1 = (int)((u1 * ctas - 1) / total);
  if (b0 == b1) return;
  const int kvh = u / s.row_tiles, rt = u - kvh * s.row_tiles;
  const int row0 = rt * a.tile_rows, rows = min(a.tile_rows, s.n * a.G - row0);
  // the unit is the second part of the CTA it begins in the middle of, the first of all others
  const int64_t part0 = (int64_t)b0 * 2 + (total * b0 / ctas >= u0 ? 0 : 1);
  const int parts = b1 - b0 + 1;
  const auto part = [&](int i) { return (i == 0 ? part0 : (int64_t)(b0 + i) * 2) * BM; };

  const int rr = threadIdx.x % J::RT, rest = threadIdx.x / J::RT;
  const int share = SHARES > 1 ? rest : 0, cb = blockIdx.y / (BM / J::RT);
  const int r = (int)(blockIdx.y % (BM / J::RT)) * J::RT + rr;
  const int col = 16 * (SHARES > 1 ? cb : cb * J::CG + rest);
  const bool live = r < rows;
  float m = -INFINITY, l = 0.f, acc[16];
  bool lack = false;                                 // of a part whose CTA gave up
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  if (live) {
#pragma unroll 4
    for (int i = share; i < parts; i += SHARES) {
      const float x = a.part_ml[part(i) + r].x;
      lack |= isnan(x);
      m = fmaxf(m, x);
    }
    const float off = m == -INFINITY ? 0.f : m;
#pragma unroll 2
    for (int i = share; i < parts; i += SHARES) {
      const float2 p = a.part_ml[part(i) + r];
      const float4* src = reinterpret_cast<const float4*>(a.part_o + part(i) * D) + col / 4 * BM + r;
      const float f = ex2(p.x - off);
      l = fmaf(p.y, f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 v = src[e * BM];
        acc[e * 4] = fmaf(v.x, f, acc[e * 4]);
        acc[e * 4 + 1] = fmaf(v.y, f, acc[e * 4 + 1]);
        acc[e * 4 + 2] = fmaf(v.z, f, acc[e * 4 + 2]);
        acc[e * 4 + 3] = fmaf(v.w, f, acc[e * 4 + 3]);
      }
    }
  }
  if constexpr (SHARES > 1) {
    s_ml[share][rr] = make_float2(lack ? __int_as_float(0x7fffffff) : m, l);
#pragma unroll
    for (int e = 0; e < 16; ++e) s_o[share][rr * 17 + e] = acc[e];
    __syncthreads();
    if (share > 0) return;
#pragma unroll
    for (int v = 0; v < SHARES; ++v) {
      lack |= isnan(s_ml[v][rr].x);
      m = fmaxf(m, s_ml[v][rr].x);
    }
    const float off = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
    for (int v = 0; v < SHARES; ++v) {
      const float f = ex2(s_ml[v][rr].x - off);
      l = fmaf(s_ml[v][rr].y, f, l);
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] = fmaf(s_o[v][rr * 17 + e], f, acc[e]);
    }
  }
  if (!live || lack) return;
  const float inv = 1.f / l;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] *= inv;
  const int nd = (row0 + r) / a.G;
  bf16* dst = a.out + ((s.start + nd) * a.HQ + kvh * a.G + row0 + r - nd * a.G) * D + col;
  *reinterpret_cast<uint4*>(dst) = pack8(acc);
  *reinterpret_cast<uint4*>(dst + 8) = pack8(acc + 8);
}

// Rows per CTA tile, by the rows of the largest tree: 16 or 32 (mma.sync; the traffic
// bounds them), 128 on tcgen05 from 33 on (32 sequences of 6144 positions and 16 nodes
// of 4 heads: 116 us with mma.sync at 64 rows, 95 here).  Head dim 256: 64 at most, with
// mma.sync (128 rows would not fit TMEM and shared memory).  More than 128 heads to a
// kv-head: a node fills no whole tile, 32.  And how many CTAs run.
static int attn_rows(int max_nodes, int G, int D) {
  const int rows = max_nodes * G;
  return rows <= 16 ? 16 : D == 256 && rows > 32 ? 64 : rows <= 32 || G > 128 ? 32 : 128;
}
static int attn_ctas(int bm, int D) { return kAttnSms * (D <= 128 && bm <= 32 ? 2 : 1); }

struct AttnSpace {
  int64_t prefix, part_o, part_ml, bytes;
};
static AttnSpace attn_space(int bm, int n_seqs, int D) {
  const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  const int64_t rows = (int64_t)attn_ctas(bm, D) * 2 * bm;
  AttnSpace s;
  s.prefix = 0;
  s.part_o = up((n_seqs + 1ll) * 8);
  s.part_ml = s.part_o + rows * D * 4;
  s.bytes = s.part_ml + rows * 8;
  return s;
}

template <int D, int BM, int BN>
static void launch_join(const AttnArgs& a, int ctas, cudaStream_t s) {
  const int row_tiles = (a.max_nodes * a.G + a.tile_rows - 1) / a.tile_rows;
  const int units = a.n_seqs * a.HKV * row_tiles;
  if ((int64_t)units * 4 < ctas)
    attention_join_kernel<D, BM, BN, 8>
        <<<dim3(units, AttnJoin<D, BM, 8>::kBlocksY), AttnJoin<D, BM, 8>::kThreads, 0, s>>>(a, row_tiles, ctas);
  else
    attention_join_kernel<D, BM, BN, 1>
        <<<dim3(units, AttnJoin<D, BM, 1>::kBlocksY), AttnJoin<D, BM, 1>::kThreads, 0, s>>>(a, row_tiles, ctas);
}

template <int D, int WM, int WN>
static int launch_attention(const CUtensorMap& kmap, const CUtensorMap& vmap, const AttnArgs& a,
                            cudaStream_t s) {
  using P = Attn<D, WM, WN>;
  constexpr size_t bytes = sizeof(typename P::Smem) + 1024;
  static_assert((bytes + 1024) * P::CTAS <= 228 * 1024, "shared memory of one SM");
  auto fn = attention_tree_kernel<D, WM, WN>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
      cudaSuccess)
    return check_launch("gdn_attention_tree");
  const int ctas = attn_ctas(P::BM, D);
  fn<<<ctas, 32 * (P::NC + 1), bytes, s>>>(kmap, vmap, a);
  if (a.max_len > P::BN) launch_join<D, P::BM, P::BN>(a, ctas, s);   // else no unit is cut
  return check_launch("gdn_attention_tree");
}

template <int D>
static int launch_attention_tc(const CUtensorMap& kmap, const CUtensorMap& vmap,
                               const CUtensorMap& qmap, const AttnArgs& a, cudaStream_t s) {
  using P = AttnTc<D>;
  constexpr size_t bytes = sizeof(typename P::Smem) + 1024;
  static_assert(bytes + 1024 <= 228 * 1024, "shared memory of one SM");
  auto fn = attention_tree_tc_kernel<D>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
      cudaSuccess)
    return check_launch("gdn_attention_tree");
  const int ctas = attn_ctas(P::BM, D);
  fn<<<ctas, 384, bytes, s>>>(kmap, vmap, qmap, a);
  if (a.max_len > P::BN) launch_join<D, P::BM, P::BN>(a, ctas, s);   // else no unit is cut
  return check_launch("gdn_attention_tree");
}

}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_attention_tree_workspace_bytes(int32_t n_seqs, int32_t num_q_heads,
                                                      int32_t num_kv_heads, int32_t head_dim,
                                                      int32_t max_nodes) {
  if (n_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_nodes <= 0)
    return 0;
  return attn_space(attn_rows(max_nodes, num_q_heads / num_kv_heads, head_dim), n_seqs,
                    head_dim).bytes;
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
  GDN_REQUIRE(scale > 0.f && scale < 1e30f, "%s: the scale must be positive", fn);
  GDN_REQUIRE(q && k_cache && v_cache && block_tables && context_lens && cu_seqlens && parents && out,
              "%s: null pointer", fn);
  GDN_REQUIRE(num_blocks > 0 && max_blocks > 0, "%s: no pages", fn);
  GDN_UNSUPPORTED(((q_row_stride | block_stride | token_stride | head_stride) & 7) == 0 &&
                      aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out),
                  "%s: operands and strides must be 16-byte aligned", fn);
  const int G = num_q_heads / num_kv_heads, bm = attn_rows(max_nodes, G, head_dim);
  const int tile_rows = bm == 128 ? 128 / G * G : bm;
  // the scan adds up 32-bit tile counts of up to 384 sequences; TMA coordinates are 32 bits
  const int row_tiles = (max_nodes * G + tile_rows - 1) / tile_rows;
  GDN_UNSUPPORTED((max_len / 64 + 1ll) * num_kv_heads * row_tiles <= (1ll << 22) &&
                      num_blocks < (1ll << 31) && max_len <= (1 << 30) && n_tokens < (1ll << 31),
                  "%s: max_len %d with %d kv heads too large", fn, max_len, num_kv_heads);
  GDN_UNSUPPORTED((int64_t)n_seqs * num_kv_heads * row_tiles < (1ll << 31),
                  "%s: too many sequences or heads", fn);
  const AttnSpace sp = attn_space(bm, n_seqs, head_dim);
  GDN_REQUIRE(workspace != nullptr && workspace_bytes >= sp.bytes && aligned16(workspace),
              "%s: workspace of %lld bytes needed (16-byte aligned), got %lld", fn,
              (long long)sp.bytes, (long long)workspace_bytes);
  int box = 64;                                    // positions per TMA box: divides a page
  while (block_size % box) box /= 2;
  const EncodeTiledFn encode = encode_tiled();
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)num_kv_heads, (cuuint64_t)block_size,
                              (cuuint64_t)num_blocks};
  const cuuint64_t strides[3] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2,
                                 (cuuint64_t)block_stride * 2};
  const cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1}, step[4] = {1, 1, 1, 1};
  // fetches into L2 no wider than a position's head: with 256 bytes, head dim 64 read half of
  // its neighbour heads' data too, long before they were wanted (444 MB where 302 are needed)
  const auto promotion = head_dim == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                        : CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
  CUtensorMap kmap, vmap;
  const auto make = [&](CUtensorMap* m, const void* p) {
    return encode != nullptr &&
           encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, boxes,
                  step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, promotion,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (!make(&kmap, k_cache) || !make(&vmap, v_cache)) {
    set_error("%s: the caches' tensor maps could not be encoded", fn);
    return GDN_ERR_CUDA;
  }
  char* ws = static_cast<char*>(workspace);
  const AttnArgs a{(const bf16*)q, q_row_stride, num_blocks, block_size, box, block_tables,
                   table_stride, max_blocks, context_lens, cu_seqlens, n_seqs, parents, max_nodes,
                   n_tokens, max_len, (bf16*)out, num_q_heads, num_kv_heads, G, tile_rows,
                   scale * 1.4426950408889634f, reinterpret_cast<int64_t*>(ws + sp.prefix),
                   reinterpret_cast<float*>(ws + sp.part_o),
                   reinterpret_cast<float2*>(ws + sp.part_ml), wait_limit(kAttnWait), status};
  cudaStream_t s = (cudaStream_t)stream;
#define GDN_AT(D)                                                    \
  if (bm == 16) return launch_attention<D, 1, 4>(kmap, vmap, a, s);  \
  if (bm == 32) return launch_attention<D, 2, 2>(kmap, vmap, a, s);
  if (head_dim == 64) { GDN_AT(64) }
  if (head_dim == 128) { GDN_AT(128) }
  if (head_dim == 256) { GDN_AT(256) }
#undef GDN_AT
  if (head_dim == 256) return launch_attention<256, 4, 1>(kmap, vmap, a, s);
  // whole nodes of a group's heads: one box brings a row tile's queries in row order
  const cuuint64_t qdims[3] = {(cuuint64_t)head_dim, (cuuint64_t)num_q_heads, (cuuint64_t)n_tokens};
  const cuuint64_t qstrides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)q_row_stride * 2};
  const cuuint32_t qbox[3] = {64, (cuuint32_t)G, (cuuint32_t)(tile_rows / G)};
  CUtensorMap qmap;
  if (encode(&qmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), qdims, qstrides, qbox,
             step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
    set_error("%s: the queries' tensor map could not be encoded", fn);
    return GDN_ERR_CUDA;
  }
  return head_dim == 64 ? launch_attention_tc<64>(kmap, vmap, qmap, a, s)
                        : launch_attention_tc<128>(kmap, vmap, qmap, a, s);
}
