// Tree attention on the tensor cores: two CTAs of a cluster work on 128 query rows of a request.
//
// The query rows of a request (node-major: row = node * heads + head) are cut into groups of 128; a
// cluster walks a contiguous range of 128-token tiles for one group, 64 rows per CTA:
//   S[128 rows, 128 tokens] = Q . K^T        tcgen05 cta_group::2, M = 128, K-major operands
//   softmax per row, base 2, lazy rescale
//   O[128 rows, rank]      += P . V          cta_group::2, M = 128, N = 256 dims, V MN-major
// Why a pair.  32-bit accumulators of 768 output dims for 128 rows do not fit one SM's 512 TMEM
// columns; of 64 rows they take 384 (a paired M = 128 tile keeps 64 rows per CTA, the first half of N
// in lanes 0-63 and the second in lanes 64-127) and leave room for two S buffers.  And each CTA
// supplies half of every B operand - K of 64 of the tile's tokens, V of half of the output dims - so
// a byte brought into an SM serves 128 rows, not 64.  Q of 64 rows x 1000 dims takes 128 KB of shared
// memory in either case; what is left streams K and V through one ring of 16 KB slots in the order
// the MMAs take them: K(0), K(1), V(0), K(2), V(1), ... V is read again (from L2) because no SM can
// hold a tile's keys until its softmax is done.
// Groups of one request run side by side: cluster s * groups + g walks range s for group g, so
// the groups' loads of a tile meet in L2 and the cache crosses HBM once.
// A tile costs 63 + 24 MMAs, 3550 cycles at the dense rate whatever the rows in use (bf16; the
// e4m3 form doubles the MMAs at twice the rate), against 224 KB into each SM: up to one group the call
// is bound by HBM, beyond it by the tensor pipe and the L2-to-SM stream together.
//
// Weights P are rounded to bf16 (8 bits, one operand of the PV instruction, as in the decode kernel);
// over an FP8 cache to three e5m2 terms (at least 8 bits down to 2^-19 of the row's largest weight, the
// last of them lost below 2^-29).  The maximum, both sums and O are 32-bit.  O is divided by the sum of the
// rounded weights, so that the output is a mean of the values with weights off by 2^-9 at most: its error is
// at most 2^-9 sum_i p_i |v_i - o|, nothing where one token has all the weight; lse comes from the sum of
// the unrounded ones.  A second bf16 term would cost 24 more MMAs per tile and 16 KB of shared memory,
// one ring slot of the four that the widest rows leave.  Two terms with an e4m3 one among them are a third
// cheaper in PV over an FP8 cache but keep 3 bits or none below 2^-15, which a long faint tail behind one
// heavy token cannot afford.
// Values of drafted tokens and of the tail of the last page come from a copy with non-finite elements
// zeroed (prep kernel): a node that does not see such a token has P = 0 there, and 0 * NaN must not
// reach it; a node that sees it has S = NaN already.
//
// Measured on a B200 (peaks 1663 bf16 TFLOP/s, 6.55 TB/s): 16 requests of up to 32k tokens x 8 nodes x 24
// heads, rank 768, bf16: 453 us, 208 GF (28% of the peak, the tensor pipe 29% busy, DRAM 17%); 8 x 16 nodes
// over an FP8 cache 385 us; 16 x 4 nodes x 12 heads, rank 384: 213 us; one request of 517 tokens 37 us.
// A 16 x 8 tile takes 10.9k cycles, 4.0k of them QK MMAs and 2.3k PV.  What bounds it is the ring's round
// trip: beside Q only four 16 KB slots fit for its fourteen, and a slot comes back after about 3000 cycles
// (empty wait, four boxes, the copy, the MMAs).  FP8 has three slots for seven; at rank 384 eight of eight fit and
// a tile still takes about 8000 cycles: the 48 rows are all CTA 0's, and the softmax and factor work of
// empty rows is done too.
//
// Warps of a CTA: 0-7 softmax and epilogue (a thread owns 32 tokens of one row), 8-10 score factors
// (1 / rms per token and head), 11 MMA issue (leader) or the announcement that Q has landed (peer), 12-15 TMA loads,
// a slot each in turn: a warp spends 400 cycles or more on a slot's boxes (16-token pages: four of 4 KB,
// ~50 cycles each past the first); one warp for all slots would be the bound itself.
#pragma once
#include "qmla_decode.cuh"
#include "qmla_pair.cuh"
#include "qmla_qimage.cuh"

namespace qmla {

__device__ int g_tree_status;  // bits of every call that failed on this device (qmla_operator_status)

struct TreeArgs {
  const uint8_t *q, *q_pe;
  int64_t q_sr, q_sh, qpe_sr, qpe_sh;  // elements
  int q_dtype;
  const uint8_t* cache;
  int64_t page_b, tok_b, num_pages;
  const int32_t* bt;
  int64_t bt_stride, bt_cols;
  int page_size;
  const int32_t* ctx;
  const int64_t* mask;
  int64_t mask_stride;  // elements between requests; 0: one tree for all
  int reqs, nodes, heads, rank, qk_dim, rms_mode;
  int64_t rms_off_b;
  float sm_scale, logit_cap;
  const float* k_scale;
  uint8_t* o;
  int64_t o_sr, o_sh;
  int o_dtype;
  uint8_t* lse;
  int64_t lse_sr;
  int lse_dtype;
  float* part_o;    // [nsplit][rows][heads][rank]
  float* part_lse;  // [nsplit][rows][heads], log2 units
  int nsplit;
};

// Committed tokens of request r, clamped to what its block-table row can hold.
__device__ __forceinline__ int tree_ctx(const TreeArgs& a, int r) {
  const int64_t room = a.bt_cols * a.page_size;
  return (int)min((int64_t)max(__ldg(a.ctx + r), 0), room);
}

constexpr int kTrSoftWarps = 8, kTrFacWarp = 8, kTrFacWarps = 3, kTrMmaWarp = 11, kTrLoadWarp = 12, kTrLoadWarps = 4;
constexpr int kTrThreads = 512;
constexpr int kTrSoft = 32 * kTrSoftWarps;  // softmax threads
constexpr int kTrRows = 64;          // query rows per CTA
constexpr int kTrTail = 256;         // tokens of a request's copied tail (127 + 64 at most)
constexpr int kTrFacPitch = 132;     // floats between heads in the factor table
constexpr int kTrMaxSlots = 10;
constexpr uint32_t kTrSlot = 16384;
constexpr int tr_p_bytes(bool fp8) { return fp8 ? 24576 : 16384; }  // P of a CTA's 64 rows x 128 tokens

// Instruction descriptor of a paired M = 128 tile: 32-bit sums, A K-major, formats 0 = e4m3 (f16),
// 1 = e5m2 (bf16); b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t tr_idesc(uint32_t fa, uint32_t fb, uint32_t N, uint32_t b_mn) {
  return (1u << 4) | (fa << 7) | (fb << 10) | (b_mn << 16) | ((N >> 3) << 17) | ((128u >> 4) << 24);
}

struct TreeMma {
  int32_t* prefix;   // [reqs + 1] tiles
  int32_t* bounds;   // [ranges + 1]
  uint8_t* img;      // [reqs][groups][2][img_bytes]
  float* q_inv;      // [reqs][groups][128] inverse query scalings (FP8)
  uint8_t* tail;     // [reqs][kTrTail][rank]
  float* part_o;     // [2 * ranges][groups][128][rank]
  float* part_lse;   // [2 * ranges][groups][128], log2 units
  int* status;               // of this call
  uint32_t wait_us;          // how long a wait may last
  int groups, ranges, rows;  // rows = nodes * heads
  int terms, chunks, full_chunks, v_chunks;
  int run;                   // tokens per K / V box
  int seg_cost;
  uint32_t img_bytes, nslots, off_q, off_p, off_fac, off_misc;
  int units, base_b, skip;   // rms tail: 16-byte units per token, first byte, bytes to skip
  int o_cols;                // TMEM columns of O
  int o_vec, q_vec;          // 16-byte accesses of o / q are legal
};
struct TreeMaps {
  CUtensorMap chunk;  // (element, token in page, page), box = one 128-byte column x run tokens
  CUtensorMap wide;   // (element, token in group, column, group in page, page), box = 2 columns x run
  CUtensorMap tail;   // (element, token), box = one 128-byte column x 64 tokens
};

// Tokens of request r: committed and drafted, within its block-table row.
__device__ __forceinline__ int64_t tree_tokens(const TreeArgs& a, int r) {
  return min((int64_t)tree_ctx(a, r) + a.nodes, a.bt_cols * a.page_size);
}

// Query images, the sanitised tail, the tile prefix and range bounds.  A warp per image row, then a
// warp per tail token; the last block plans.
template <bool FP8>
__global__ void __launch_bounds__(256) tree_prep_kernel(const TreeArgs a, const TreeMma m) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t qrows = (int64_t)a.reqs * m.groups * 128, trows = (int64_t)a.reqs * kTrTail;
  if (blockIdx.x + 1 < gridDim.x) {
    int64_t w = (int64_t)blockIdx.x * 8 + warp;
    if (w < qrows) {
      const int r = (int)(w / (m.groups * 128)), x = (int)(w - (int64_t)r * m.groups * 128);
      const int node = x / a.heads, h = x - node * a.heads;
      const QSource s{a.q, a.q_pe, a.q_sr, a.q_sh, a.qpe_sr, a.qpe_sh, a.q_dtype, a.rank, a.qk_dim, m.q_vec};
      uint8_t* img = m.img + (w >> 6) * m.img_bytes;  // 64 rows per image
      const float inv = write_q_row<FP8>(s, x < m.rows ? (int64_t)r * a.nodes + node : -1, h, img, x & 63, kTrRows,
                                         m.chunks, m.terms);
      if (lane == 0) m.q_inv[w] = inv;
      return;
    }
    w -= qrows;
    if (w >= trows) return;
    const int r = (int)(w / kTrTail), i = (int)(w - (int64_t)r * kTrTail);
    const int64_t n = tree_tokens(a, r), t = tree_ctx(a, r) / kTile * kTile + i;
    if (t / kTile >= (n + kTile - 1) / kTile) return;  // no such tile
    const uint8_t* src = nullptr;
    if (t < n) {
      const int pg = __ldg(a.bt + r * a.bt_stride + t / a.page_size);
      if (pg >= 0 && pg < a.num_pages) src = a.cache + (int64_t)pg * a.page_b + t % a.page_size * a.tok_b;
    }
    const int units = a.rank * (FP8 ? 1 : 2) / 16;
    uint4* dst = reinterpret_cast<uint4*>(m.tail + w * a.rank * (FP8 ? 1 : 2));
    for (int u = lane; u < units; u += 32) {
      uint4 v = src ? __ldg(reinterpret_cast<const uint4*>(src) + u) : make_uint4(0u, 0u, 0u, 0u);
      uint32_t* e = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (FP8) {
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if ((e[k] >> (8 * b) & 0x7f) == 0x7f) e[k] &= ~(0xffu << (8 * b));
        } else {
          if ((e[k] & 0x7f80u) == 0x7f80u) e[k] &= 0xffff0000u;
          if ((e[k] & 0x7f800000u) == 0x7f800000u) e[k] &= 0x0000ffffu;
        }
      }
      dst[u] = v;
    }
    return;
  }
  __shared__ int warp_sum[8];
  __shared__ int carry;
  if (threadIdx.x == 0) {
    carry = 0;
    m.prefix[0] = 0;
    *m.status = 0;
  }
  for (int base = 0; base < a.reqs; base += 256) {
    const int i = base + threadIdx.x;
    int x = i < a.reqs ? (int)((tree_tokens(a, i) + kTile - 1) / kTile) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    x += carry;
    for (int w = 0; w < warp; ++w) x += warp_sum[w];
    if (i < a.reqs) m.prefix[i + 1] = x;
    __syncthreads();
    if (threadIdx.x == 255) carry = x;
  }
  __threadfence_block();
  __syncthreads();
  for (int c = threadIdx.x; c <= m.ranges; c += 256) m.bounds[c] = range_bound(m.prefix, a.reqs, m.ranges, m.seg_cost, c);
}

// TERMS: terms of a query element (qmla_qimage.cuh).
template <bool FP8, int TERMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTrThreads, 1)
    tree_mma_kernel(const __grid_constant__ TreeMaps maps, const TreeArgs a, const TreeMma m) {
  constexpr float kThr = FP8 ? 2.f : 8.f;    // log2 units a weight may exceed 1 by before O is rescaled
  constexpr float kShift = FP8 ? 13.f : 0.f;  // P = 2^(x - m + shift), up to 2^15 where e5m2 ends
  constexpr int kPTerms = FP8 ? 3 : 1;
  constexpr int es = FP8 ? 1 : 2;
  constexpr int E = 128 / es;                // elements of a 128-byte column
  constexpr int NV = FP8 ? 1 : 2;            // token halves of a V tile held in slots of their own
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_rank();
  const int cluster = blockIdx.x >> 1;
  const int range = cluster / m.groups, g = cluster - range * m.groups;
  const int lo = __ldg(m.bounds + range), hi = __ldg(m.bounds + range + 1);
  if (lo >= hi) return;  // the same for both CTAs
  const int req0 = first_row_at(m.prefix, a.reqs, lo);

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + m.off_misc);
  // leader's: full (both CTAs' loads of a slot), sempty, pfull, ofree, qpeer.  Each CTA's own: empty,
  // sfull, odone, qempty (all arrived on by the leader's commits), qfull, facfull, facfree.
  const uint32_t b_full = 0, b_empty = m.nslots, b_sfull = 2 * m.nslots, b_sempty = b_sfull + 2, b_pfull = b_sempty + 2,
                 b_odone = b_pfull + 1, b_ofree = b_odone + 1, b_qfull = b_ofree + 1, b_qempty = b_qfull + 1,
                 b_qpeer = b_qempty + 1, b_facfull = b_qpeer + 1, b_facfree = b_facfull + 1, b_fin = b_facfree + 1,
                 n_bars = b_fin + 1;
  auto bar = [&](uint32_t i) { return smem_u32(bars + i); };
  auto leader = [&](uint32_t i) { return map_cta(smem_u32(bars + i), 0); };
  uint8_t* misc = reinterpret_cast<uint8_t*>(bars + n_bars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + 4);
  volatile uint32_t* valid_s = reinterpret_cast<volatile uint32_t*>(misc + 16);  // [4] tokens that exist
  float* red = reinterpret_cast<float*>(misc + 32);                              // [4][64]
  float* fac = reinterpret_cast<float*>(smem + m.off_fac);                       // [heads][kTrFacPitch]
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < m.nslots; ++i) {
      mbar_init(bar(b_full + i), 1);
      mbar_init(bar(b_empty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(b_sfull + i), 1);
      mbar_init(bar(b_sempty + i), 2 * kTrSoftWarps);
    }
    mbar_init(bar(b_pfull), 2 * kTrSoftWarps);
    mbar_init(bar(b_odone), 1);
    mbar_init(bar(b_ofree), 2 * kTrSoftWarps);
    mbar_init(bar(b_qfull), 1);
    mbar_init(bar(b_qempty), 1);
    mbar_init(bar(b_qpeer), 1);
    mbar_init(bar(b_facfull), kTrFacWarps);
    mbar_init(bar(b_facfree), kTrSoftWarps);
    mbar_init(bar(b_fin), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kTrMmaWarp) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are ready
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t col_s = m.o_cols;
  const uint32_t qbuf = sbase + m.off_q, pbuf = sbase + m.off_p;
  const int v_blocks = (m.v_chunks + 2 * NV - 1) / (2 * NV);  // 256-dim output blocks
  // 128-byte V columns of block nb that CTA c holds: FP8 one (none past the rank), bf16 two, or
  // one in a last block of 128 dims
  auto v_cols = [&](int nb, int c) -> int {
    if constexpr (FP8) return 2 * nb + c < m.v_chunks ? 1 : 0;
    return m.v_chunks - 4 * nb >= 4 ? 2 : 1;
  };
  auto v_col0 = [&](int nb, int c) -> int { return FP8 ? 2 * nb + c : 4 * nb + c * v_cols(nb, c); };

  if (warp >= kTrLoadWarp) {
    // ---------------------------------------------------------------- loads
    // The load warps take the slots in turn (no more warps than slots: a warp then filled the slot
    // `warps` before this one, so the phase it waits for is never two behind).  All lanes wait; lane 0
    // arms the leader's barrier for both CTAs' bytes; each of the first lanes issues one box.  What a
    // box needs beside its column is worked out once per tile.
    const uint32_t lw = warp - kTrLoadWarp, nlw = min((uint32_t)kTrLoadWarps, m.nslots);
    uint32_t turn = lw < nlw ? 0u : 1000u;  // whose slot is next (a warp without slots never matches)
    const uint64_t pol = policy_evict_normal();
    const int run = m.run, khalf = 64 / run;  // boxes of a CTA's 64 tokens of K
    const int k_slots = (m.chunks + 1) / 2;
    const uint32_t full0 = leader(b_full);
    const int kb = lane % khalf, kc = lane / khalf;        // this lane's K box: run, column (plain slots)
    const int vbox = (kTile / NV) / run, vb = lane % vbox;  // V boxes of a slot, this lane's
    const uint32_t k_wide = kb * run * 256, k_plain = kc * 8192 + kb * run * 128;
    SegCursor cur{req0, lo, hi};
    int r, k0, k1, plo, phi;
    uint32_t seg = 0, count = 0;  // slots so far
    Ring ring;
    bool ok = true;
    auto slot_mine = [&]() { return turn == lw; };
    auto slot_next = [&]() {
      ring.next(m.nslots);
      ++count;
      if (lw < nlw) turn = turn + 1 == nlw ? 0u : turn + 1;
    };
    auto slot_begin = [&](uint32_t bytes) {
      ok = mbar_wait_for(bar(b_empty + ring.idx), ring.ph ^ 1, abort_flag, m.status, m.wait_us);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && cta == 0 && lane == 0) mbar_expect_tx(bar(b_full + ring.idx), bytes);
    };
    while (ok && next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
      if (lw == 0) {
        if (seg > 0) ok = mbar_wait_for(bar(b_qempty), (seg - 1) & 1, abort_flag, m.status, m.wait_us);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(bar(b_qfull), m.img_bytes);
          load_image(qbuf, m.img + (((int64_t)r * m.groups + g) * 2 + cta) * m.img_bytes, m.img_bytes, bar(b_qfull), pol);
        }
      }
      ++seg;
      const int n = (int)tree_tokens(a, r);
      const int tail_tile = tree_ctx(a, r) / kTile;
      const int32_t* bt = a.bt + r * a.bt_stride;
      int pg_next = -1, y_next = 0;  // page (-1 past the end) and row in it of token run `lane` of a tile
      auto look_up = [&](int k) {
        const uint32_t tok = (uint32_t)k * kTile + lane * run;
        pg_next = -1;
        if (lane < 2 * khalf && tok < (uint32_t)n) {
          const uint32_t pi = tok / (uint32_t)a.page_size;
          y_next = (int)(tok - pi * (uint32_t)a.page_size);
          pg_next = __ldg(bt + pi);
        }
      };
      look_up(k0);
      int pg_prev = -1, y_prev = 0;
      for (int k = k0; k <= k1 && ok; ++k) {
        const int pg = pg_next, y = y_next;
        if (k + 1 < k1) look_up(k + 1);  // on its way during this tile
        if (k < k1) {  // K of tile k: this CTA's 64 tokens, two columns per slot
          const int kpg = __shfl_sync(0xffffffffu, pg, (int)cta * khalf + kb);
          const int ky = __shfl_sync(0xffffffffu, y, (int)cta * khalf + kb);
          for (int s = 0; s < k_slots; ++s, slot_next()) {
            if (!slot_mine()) continue;
            const int c0 = 2 * s, nch = min(2, m.chunks - c0);
            slot_begin((uint32_t)nch * 2u * 8192u);
            if (!ok) break;
            const uint32_t slot = sbase + ring.idx * kTrSlot, fb = full0 + ring.idx * 8;
            if (c0 + 2 > m.full_chunks) {
              if (kc < nch) tma_load_3d_pair(slot + k_plain, &maps.chunk, (c0 + kc) * E, ky, kpg, fb, pol);
            } else if (lane < khalf) {
              tma_load_5d_pair(slot + k_wide, &maps.wide, 0, 0, c0, ky >> 3, kpg, fb, pol);
            }
          }
        }
        if (k > k0 && ok) {  // V of tile k - 1: all its tokens, this CTA's half of the dims
          const int kv = k - 1;
          const bool tail = kv >= tail_tile;
          const int row0 = r * kTrTail + (kv - tail_tile) * kTile;  // in the copied tail
          for (int th = 0; th < NV && ok; ++th) {
            const int vpg = __shfl_sync(0xffffffffu, pg_prev, th * khalf + vb);
            const int vy = __shfl_sync(0xffffffffu, y_prev, th * khalf + vb);
            for (int nb = 0; nb < v_blocks; ++nb, slot_next()) {
              if (!slot_mine()) continue;
              const int nc = v_cols(nb, (int)cta), vc0 = v_col0(nb, (int)cta);
              constexpr int toks = kTile / NV;
              slot_begin((uint32_t)((v_cols(nb, 0) + v_cols(nb, 1)) * toks * 128));
              if (!ok) break;
              const uint32_t slot = sbase + ring.idx * kTrSlot, fb = full0 + ring.idx * 8;
              if (tail) {
                if (lane < nc * (toks / 64)) {
                  const int cc = NV == 2 ? lane : 0, tb = NV == 2 ? 0 : lane;
                  tma_load_2d_pair(slot + lane * 8192, &maps.tail, (vc0 + cc) * E, row0 + th * 64 + tb * 64, fb, pol);
                }
              } else if (lane < vbox && nc > 0) {
                if (nc == 2)
                  tma_load_5d_pair(slot + lane * run * 256, &maps.wide, 0, 0, vc0, vy >> 3, vpg, fb, pol);
                else
                  tma_load_3d_pair(slot + lane * run * 128, &maps.chunk, vc0 * E, vy, vpg, fb, pol);
              }
            }
          }
        }
        pg_prev = pg;
        y_prev = y;
      }
    }
    if (!ok && lane == 0) {  // after an abort: wait (bounded) for the copies already issued
      volatile int never = 0;
      if (cta == 0 && lw < nlw)
        for (uint32_t p = count > m.nslots ? count - m.nslots : 0u; p < count; ++p)
          if (p % nlw == lw) mbar_wait(bar(b_full + p % m.nslots), (p / m.nslots) & 1, &never, nullptr, 20000000ull);
      if (lw == 0 && seg > 0) mbar_wait(bar(b_qfull), (seg - 1) & 1, &never, nullptr, 20000000ull);
      // The peer's copies report to the leader's barriers, which may not even be armed for them when the
      // leader gave up first: 1 ms, hundreds of times what a copy takes, lets them land.
      if (cta == 1)
        for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 1000000ull;) __nanosleep(2000);
    }
    __syncwarp();
  } else if (warp == kTrMmaWarp) {
    // ---------------------------------------------------------------- MMA issue
    SegCursor cur{req0, lo, hi};
    int r, k0, k1, plo, phi;
    uint32_t seg = 0;
    bool ok = true;
    if (cta == 1) {  // tell the leader that this CTA's Q has landed
      while (ok && next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
        ok = __all_sync(0xffffffffu, mbar_wait_for(bar(b_qfull), seg & 1, abort_flag, m.status, m.wait_us));
        if (ok && lane == 0) mbar_arrive_cluster(leader(b_qpeer));
        ++seg;
      }
    } else {
      const uint32_t q_lo = sdesc_lo(qbuf, 16), p_lo = sdesc_lo(pbuf, 16);
      const uint32_t qt16 = (uint32_t)(m.chunks * kTrRows * 128) >> 4;
      const uint32_t slot0 = sbase >> 4;
      const int k_slots = (m.chunks + 1) / 2;
      uint32_t js = 0, jp = 0;  // tiles scored / accumulated so far
      Ring ring;
      auto wait = [&](uint32_t b, uint32_t ph) {  // the whole warp
        ok = ok && mbar_wait_for(bar(b), ph, abort_flag, m.status, m.wait_us);
        ok = __all_sync(0xffffffffu, ok);
      };
      // The slot at the head of the ring.  Its barrier is tried before the MMAs of the slot before it
      // are issued, so that the answer is there when they are.
      bool peek = false;
      auto slot_wait = [&]() {
        if (!__all_sync(0xffffffffu, peek)) wait(b_full + ring.idx, ring.ph);
        tc_fence_after();
      };
      auto slot_peek_next = [&]() {
        Ring nx = ring;
        nx.next(m.nslots);
        peek = mbar_try_wait(bar(b_full + nx.idx), nx.ph);
      };
      auto slot_done = [&]() {
        tc_commit_pair(bar(b_empty + ring.idx));
        ring.next(m.nslots);
      };
      auto qk = [&]() {
        const uint32_t sb = js & 1;
        if (js >= 2) wait(b_sempty + sb, ((js - 2) >> 1) & 1);
        const uint32_t d = tmem + col_s + sb * 64;
        uint32_t a_lo = q_lo;
        for (int s = 0; s < k_slots; ++s, a_lo += 2 * kTrRows * 128 >> 4) {
          slot_wait();
          if (!ok) return;
          slot_peek_next();
          // column ci of the slot: 8 KB on (plain), or between the 8-row groups
          const bool plain = 2 * s + 2 > m.full_chunks;
          const uint32_t b_lo = slot0 + ring.idx * (kTrSlot >> 4) + (1u << 16), b_hi = plain ? sdesc_hi(1024) : sdesc_hi(2048);
          const uint32_t b_col = plain ? 8192 >> 4 : 1024 >> 4;
          const bool two = 2 * s + 1 < m.chunks;
#pragma unroll
          for (int ci = 0; ci < 2; ++ci) {
            if (ci == 0 || two) {
#pragma unroll
              for (int t = 0; t < TERMS; ++t) {
                constexpr uint32_t id0 = tr_idesc(0, 0, 128, 0), id1 = tr_idesc(1, 0, 128, 0), idb = tr_idesc(1, 1, 128, 0);
                const uint32_t al = a_lo + ci * (kTrRows * 128 >> 4) + t * qt16, bl = b_lo + ci * b_col;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                  tc_mma_pair<FP8>(d, al + ks * 2, sdesc_hi(1024), bl + ks * 2, b_hi, !FP8 ? idb : t == 0 ? id0 : id1,
                                   ci + t + ks > 0 ? 1u : (uint32_t)s);
              }
            }
          }
          slot_done();
        }
        tc_commit_pair(bar(b_sfull + sb));
        ++js;
      };
      while (ok && next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
        wait(b_qfull, seg & 1);
        wait(b_qpeer, seg & 1);
        if (!ok) break;
        const int tail_tile = tree_ctx(a, r) / kTile;
        qk();
        for (int k = k0; k < k1 && ok; ++k) {
          if (k + 1 < k1)
            qk();
          else
            tc_commit_pair(bar(b_qempty));  // Q is free once the segment's scores are done
          wait(b_pfull, jp & 1);
          if (k == k0 && seg > 0) wait(b_ofree, (seg - 1) & 1);
          const bool tail = k >= tail_tile;
          const uint32_t acc0 = k > k0;
          for (int th = 0; th < NV && ok; ++th)
            for (int nb = 0; nb < v_blocks; ++nb) {
              slot_wait();
              if (!ok) break;
              // (the slot after a segment's last V belongs to the next segment's K: not tried here)
              if (th + 1 < NV || nb + 1 < v_blocks || k + 1 < k1)
                slot_peek_next();
              else
                peek = false;
              const uint32_t slot = slot0 + ring.idx * (kTrSlot >> 4);
              const uint32_t d = tmem + nb * 128;
              if constexpr (FP8) {
                const uint32_t bl = slot + (8192u >> 4 << 16);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                  for (int t = 0; t < kPTerms; ++t)
                    tc_mma_pair<true>(d, p_lo + t * (8192 >> 4) + ks * 2, sdesc_hi(1024), bl + ks * (4096 >> 4), sdesc_hi(1024),
                                      tr_idesc(1, 0, 256, 1), ks + t > 0 ? 1u : acc0);
              } else {
                const int nc = v_cols(nb, 0);
                const uint32_t id = nc == 2 ? tr_idesc(1, 1, 256, 1) : tr_idesc(1, 1, 128, 1);
                // columns of the slot LBO apart, 8-token groups SBO apart; a step is 16 tokens
                const bool paired = nc == 2 && !tail;
                const uint32_t bl = slot + (paired ? 1024u >> 4 << 16 : 8192u >> 4 << 16);
                const uint32_t bh = paired ? sdesc_hi(2048) : sdesc_hi(1024), step = paired ? 4096u >> 4 : 2048u >> 4;
                const uint32_t pl = p_lo + th * (8192 >> 4), acc1 = acc0 | (uint32_t)th;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                  tc_mma_pair<false>(d, pl + ks * 2, sdesc_hi(1024), bl + ks * step, bh, id, ks > 0 ? 1u : acc1);
              }
              slot_done();
            }
          if (ok) tc_commit_pair(bar(b_odone));
          ++jp;
        }
        ++seg;
      }
      volatile int never = 0;  // drain before TMEM is released
      __syncwarp();
      tc_commit_pair(bar(b_fin));
      mbar_wait(bar(b_fin), 0, &never, nullptr, 100000000ull);
    }
    __syncwarp();
  } else if (warp >= kTrFacWarp) {
    // ---------------------------------------------------------------- score factors
    // A work item is a 16-byte unit of one token's divisors: 8 heads (two bytes each) or 16 (one byte),
    // unpacked in registers.  A tile's units are loaded before the table is free.
    constexpr int kThreads = 32 * kTrFacWarps, kBatch = 4;
    const int ft = threadIdx.x - 32 * kTrFacWarp, fw = warp - kTrFacWarp;
    const float kscale = FP8 && a.k_scale ? __ldg(a.k_scale) : 1.f;
    const float gs = a.sm_scale * kscale * (a.logit_cap > 0.f ? 1.f : kLog2e);
    const bool two = !FP8 || a.rms_mode == 2;      // bytes per divisor
    const bool split = two && (m.skip & 1);        // raw bytes at an odd offset: a divisor may span two units
    const int items = kTile * (split ? a.heads : m.units);
    auto of_bf16 = [&](uint32_t bits) -> float {
      const float rv = __uint_as_float(bits << 16);
      return rv > 0.f ? __fdividef(gs, rv) : gs;
    };
    auto of_e4m3 = [&](uint32_t bits) -> float {
      const float rv = e4m3_to_f32((uint8_t)bits) * kscale;
      return rv > 0.f ? __fdividef(gs, rv) : gs;
    };
    auto of_log8 = [&](uint32_t bits) -> float { return gs * ex2_approx(3.0f - (float)bits * (6.0f / 255.0f)); };
    // the bytes of unit u -> the table's column t
    auto unpack = [&](const uint32_t* w, int u, int t, auto of) {
      const int h0 = 16 * u - m.skip;
      float* col = fac + h0 * kTrFacPitch + t;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if ((unsigned)(h0 + e) < (unsigned)a.heads) col[e * kTrFacPitch] = of((w[e >> 2] >> (8 * (e & 3))) & 0xffu);
    };
    SegCursor cur{req0, lo, hi};
    int r, k0, k1, plo, phi;
    uint32_t jt = 0;
    bool ok = true;
    while (ok && next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
      const int n = (int)tree_tokens(a, r);
      const int32_t* bt = a.bt + r * a.bt_stride;
      // row of token t of tile k, or null when there is none
      auto row_of = [&](int k, int t) -> const uint8_t* {
        const uint32_t tok = (uint32_t)k * kTile + t;
        if (tok >= (uint32_t)n) return nullptr;
        const uint32_t pi = tok / (uint32_t)a.page_size;
        const int pg = __ldg(bt + pi);
        if (pg < 0 || pg >= a.num_pages) return nullptr;
        return a.cache + (int64_t)pg * a.page_b + (tok - pi * (uint32_t)a.page_size) * a.tok_b;
      };
      for (int k = k0; k < k1 && ok; ++k, ++jt) {
        unsigned valid[2];  // tokens 32 fw .. and 32 (fw + 3) ..
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int t = (fw + q * kTrFacWarps) * 32 + lane;
          valid[q] = __ballot_sync(0xffffffffu, t < kTile && row_of(k, t) != nullptr);
        }
        uint4 v[kBatch];
        auto load = [&](int i0) {
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int i = i0 + b * kThreads + ft;
            v[b] = make_uint4(0u, 0u, 0u, 0u);
            if (i >= items || split) continue;
            const uint8_t* p = row_of(k, i & (kTile - 1));
            if (p) v[b] = __ldg(reinterpret_cast<const uint4*>(p + m.base_b) + (i >> 7));
          }
        };
        load(0);
        if (jt > 0) ok = mbar_wait_for(bar(b_facfree), (jt - 1) & 1, abort_flag, m.status, m.wait_us);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          valid_s[fw] = valid[0];
          if (fw + kTrFacWarps < 4) valid_s[fw + kTrFacWarps] = valid[1];
        }
        for (int i0 = 0; i0 < items; i0 += kBatch * kThreads) {
          if (i0 > 0) load(i0);
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int i = i0 + b * kThreads + ft;
            if (i >= items) continue;
            const int t = i & (kTile - 1), u = i >> 7;
            const uint32_t w[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
            if (split) {
              const uint8_t* p = row_of(k, t);
              if (p) p += m.base_b + m.skip + 2 * u;
              fac[u * kTrFacPitch + t] = p ? of_bf16((uint32_t)__ldg(p) | (uint32_t)__ldg(p + 1) << 8) : gs;
            } else if (two) {
              const int h0 = (16 * u - m.skip) / 2;
              float* col = fac + h0 * kTrFacPitch + t;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if ((unsigned)(h0 + e) < (unsigned)a.heads)
                  col[e * kTrFacPitch] = of_bf16((w[e >> 1] >> (16 * (e & 1))) & 0xffffu);
            } else if (a.rms_mode == 3) {
              unpack(w, u, t, of_log8);
            } else {
              unpack(w, u, t, of_e4m3);
            }
          }
        }
        if (items == 0)  // no divisors
          for (int i = ft; i < kTile * a.heads; i += kThreads) fac[(i >> 7) * kTrFacPitch + (i & (kTile - 1))] = gs;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(b_facfull));
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax and epilogue
    const int l = threadIdx.x & 127, wg = warp >> 2;  // TMEM lane; which 32 of its 64 columns
    const int i = l & 63, half = l >> 6;              // row of the CTA; half of the tile's tokens, of a block's dims
    const int quarter = 2 * half + wg;                // this thread's 32 tokens of the tile
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int x_row = g * 128 + (int)cta * 64 + i;
    const bool live = x_row < m.rows;
    const int node = live ? x_row / a.heads : 0, h = live ? x_row - node * a.heads : 0;
    const float* fac_row = fac + h * kTrFacPitch + quarter * 32;
    const bool cap = a.logit_cap > 0.f;
    const float kscale = FP8 && a.k_scale ? __ldg(a.k_scale) : 1.f;
    const uint32_t sempty0 = leader(b_sempty), pfull0 = leader(b_pfull), ofree0 = leader(b_ofree);
    const uint32_t prow = pbuf + i * 128;
    SegCursor cur{req0, lo, hi};
    int r, k0, k1, plo, phi;
    uint32_t jt = 0;
    // ok: this warp's waits so far; dead: the warps have agreed (in a group barrier) to leave
    bool ok = true, dead = false;
    while (!dead && next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
      const int ctx = tree_ctx(a, r);
      const uint64_t bits = live ? (uint64_t)__ldg(reinterpret_cast<const long long*>(a.mask) + r * a.mask_stride + node) : 0ull;
      const bool padding = bits == 0;  // bits past the nodes name no token, but such a node is no padding
      const uint64_t mask = bits & (a.nodes >= 64 ? ~0ull : (1ull << a.nodes) - 1);
      const float q_inv = FP8 ? __ldg(m.q_inv + ((int64_t)r * m.groups + g) * 128 + cta * 64 + i) : 1.f;
      float m_ref = -INFINITY, l_part = 0.f, l_round = 0.f;  // the sum of P, and of P as PV sees it
      for (int k = k0; k < k1; ++k, ++jt) {
        const uint32_t sb = jt & 1;
        float x[32];
        ok = ok && mbar_wait_for(bar(b_sfull + sb), (jt >> 1) & 1, abort_flag, m.status, m.wait_us);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          tc_fence_after();
          tmem_ld32(tmem + lane_base + col_s + sb * 64 + wg * 32, x);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(sempty0 + sb * 8);
          ok = mbar_wait_for(bar(b_facfull), jt & 1, abort_flag, m.status, m.wait_us);
          ok = __all_sync(0xffffffffu, ok);
        }
        uint32_t vis = 0;
        if (ok) {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 f = *reinterpret_cast<const float4*>(fac_row + e);
            x[e] *= f.x;
            x[e + 1] *= f.y;
            x[e + 2] *= f.z;
            x[e + 3] *= f.w;
          }
          vis = valid_s[quarter];
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(b_facfree));
        }
        if constexpr (FP8) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] *= q_inv;
        }
        if (cap) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = a.logit_cap * tanhf(x[e] / a.logit_cap) * kLog2e;
        }
        // tokens this row sees: committed ones, and drafts of its mask
        const int nc = ctx - (k * kTile + quarter * 32);  // committed tokens from this thread's first on
        if (nc < 32 || padding) {
          uint32_t see = nc <= 0 ? 0u : nc >= 32 ? ~0u : (1u << nc) - 1;
          if (nc >= 0)
            see |= nc < 32 ? (uint32_t)(mask << nc) : 0u;
          else
            see |= -nc < 64 ? (uint32_t)(mask >> -nc) : 0u;
          vis &= padding ? 0u : see;
        }
        float mx = -INFINITY;
        if (vis == ~0u) {
          float mq[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int e = 4; e < 32; ++e) mq[e & 3] = fmaxf(mq[e & 3], x[e]);
          mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (!(vis >> e & 1)) x[e] = -INFINITY;
            mx = fmaxf(mx, x[e]);
          }
        }
        bool need = mx > m_ref + kThr;
        // one group barrier per tile reduces the rescale test and any failed wait
        need = named_bar_or(1, kTrSoft, need || !ok);
        if (need) {
          dead = named_bar_or(1, kTrSoft, !ok);
          if (dead) break;
          red[quarter * 64 + i] = mx;
          named_bar_sync(1, kTrSoft);
          const float mn = fmaxf(fmaxf(fmaxf(red[i], red[64 + i]), fmaxf(red[128 + i], red[192 + i])), m_ref);
          const float al = mn == m_ref ? 1.f : m_ref == -INFINITY ? 0.f : exp2f(m_ref - mn);
          m_ref = mn;
          l_part *= al;
          l_round *= al;
          if (named_bar_or(1, kTrSoft, al != 1.f && k > k0)) {  // (red[] is free again)
            ok = mbar_wait_for(bar(b_odone), (jt - 1) & 1, abort_flag, m.status, m.wait_us);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              tc_fence_after();
              for (int c = wg * 16; c < m.o_cols; c += 32) {  // the warpgroups take every other 16 columns
                float o[16];
                tmem_ld16(tmem + lane_base + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= al;
                tmem_st16(tmem + lane_base + c, o);
              }
              tmem_wait_st();
              tc_fence_before();
            }
          }
        }
        // P = 2^(x - m): nothing where the row sees nothing, or only scores of -inf, so far (m = -inf)
        const float sub = m_ref == -INFINITY ? 0.f : m_ref - kShift;
        uint32_t w[FP8 ? 24 : 16];
        float ls[4] = {0.f, 0.f, 0.f, 0.f}, lr[4] = {0.f, 0.f, 0.f, 0.f};
        if constexpr (!FP8) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float pa = ex2_approx(x[e] - sub), pb = ex2_approx(x[e + 1] - sub);
            ls[e & 2] += pa;
            ls[(e & 2) + 1] += pb;
            const __nv_bfloat162 b = __floats2bfloat162_rn(pa, pb);
            w[e >> 1] = *reinterpret_cast<const uint32_t*>(&b);
            lr[e & 2] += __uint_as_float(w[e >> 1] << 16);
            lr[(e & 2) + 1] += __uint_as_float(w[e >> 1] & 0xffff0000u);
          }
        } else {
          // e5m2 is the upper byte of f16: P goes to f16, is rounded there to 9 significant bits, and the
          // three terms are what its upper byte holds, three bits at a time (exact subtractions).
          // A NaN's bits may wrap in the rounding; it is in l_part already.
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint32_t v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float pa = ex2_approx(x[4 * q + 2 * e] - sub), pb = ex2_approx(x[4 * q + 2 * e + 1] - sub);
              ls[2 * e] += pa;
              ls[2 * e + 1] += pb;
              const __half2 hv = __floats2half2_rn(pa, pb);
              v[e] = (*reinterpret_cast<const uint32_t*>(&hv) + 0x00020002u) & 0xfffcfffcu;
              const float2 pr = __half22float2(*reinterpret_cast<const __half2*>(&v[e]));
              lr[2 * e] += pr.x;
              lr[2 * e + 1] += pr.y;
            }
#pragma unroll
            for (int t = 0; t < kPTerms; ++t) {
              w[8 * t + q] = __byte_perm(v[0], v[1], 0x7531);  // the upper bytes of four values
              if (t + 1 < kPTerms) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t top = v[e] & 0xff00ff00u;
                  const __half2 rest = __hsub2(*reinterpret_cast<const __half2*>(&v[e]), *reinterpret_cast<const __half2*>(&top));
                  v[e] = *reinterpret_cast<const uint32_t*>(&rest);
                }
              }
            }
          }
        }
        l_part += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        l_round += (lr[0] + lr[1]) + (lr[2] + lr[3]);
        // the P buffer is free, and O at rest, once the previous tile's PV is done
        if (ok && jt > 0) ok = mbar_wait_for(bar(b_odone), (jt - 1) & 1, abort_flag, m.status, m.wait_us);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          if constexpr (!FP8) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              st_shared_v4(prow + half * 8192 + (((wg * 4 + u) ^ (i & 7)) << 4), w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
          } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t at = prow + (((quarter * 2 + u) ^ (i & 7)) << 4);
#pragma unroll
              for (int t = 0; t < kPTerms; ++t)
                st_shared_v4(at + t * 8192, w[8 * t + 4 * u], w[8 * t + 4 * u + 1], w[8 * t + 4 * u + 2], w[8 * t + 4 * u + 3]);
            }
          }
          fence_proxy_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(pfull0);
        }
      }
      if (dead) break;
      // ---- O / l -> the output, or this range's piece of it
      ok = ok && mbar_wait_for(bar(b_odone), (jt - 1) & 1, abort_flag, m.status, m.wait_us);
      red[quarter * 64 + i] = l_part;
      dead = named_bar_or(1, kTrSoft, !ok);
      if (dead) break;
      tc_fence_after();
      const float lt = (red[i] + red[64 + i]) + (red[128 + i] + red[192 + i]);
      named_bar_sync(1, kTrSoft);
      red[quarter * 64 + i] = l_round;
      named_bar_sync(1, kTrSoft);
      const float lr = (red[i] + red[64 + i]) + (red[128 + i] + red[192 + i]);
      const float inv = lt == 0.f ? 0.f : lt != lt ? lt : kscale / lr;
      const bool full = plo >= lo && phi <= hi;
      const int64_t piece = ((int64_t)(plo <= lo ? 2 * range : 2 * range + 1) * m.groups + g) * 128 + cta * 64 + i;
      const int64_t orow = (int64_t)r * a.nodes + node;
      uint8_t* op = a.o + (orow * a.o_sr + (int64_t)h * a.o_sh) * dt_size(a.o_dtype);
      for (int nb = 0; nb < v_blocks; ++nb) {
        const int cols = FP8 ? 128 : 64 * v_cols(nb, 0);  // dims of this block in a lane
        const int d0 = nb * 256 + half * cols;
        for (int c = wg * 16; c < cols; c += 32) {
          float o[16];
          tmem_ld16(tmem + lane_base + nb * 128 + c, o);
          tmem_wait_ld();
          if (!live || d0 + c >= a.rank) continue;
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = lt == 0.f ? 0.f : o[e] * inv;
          if (!full) {
            float4* p = reinterpret_cast<float4*>(m.part_o + piece * a.rank + d0 + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          } else if (a.o_dtype == 0 && m.o_vec) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(o[2 * e], o[2 * e + 1]);
              pk[e] = *reinterpret_cast<const uint32_t*>(&b);
            }
            uint4* p = reinterpret_cast<uint4*>(op + (int64_t)(d0 + c) * 2);
            p[0] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            p[1] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              store_from_float(op + (int64_t)(d0 + c + e) * dt_size(a.o_dtype), a.o_dtype, o[e]);
          }
        }
      }
      if (live && quarter == 0) {
        const float l2 = lt == 0.f ? -INFINITY : m_ref + log2f(lt) - kShift;
        if (!full)
          m.part_lse[piece] = l2;
        else if (a.lse)
          store_from_float(a.lse + (orow * a.lse_sr + h) * dt_size(a.lse_dtype), a.lse_dtype, l2 * kLn2);
      }
      tc_fence_before();
      named_bar_sync(1, kTrSoft);  // red[] is read
      if (lane == 0) mbar_arrive_cluster(ofree0);
    }
  }
  // ---------------------------------------------------------------- teardown
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // neither CTA leaves while the other may still signal it or read its tiles
  if (warp == kTrMmaWarp) {
    // The leader has seen its own arrival of the last commit (b_fin).  The peer's may still be on its way
    // here, and so may those of the commits before it: this CTA's barriers stay until it is there.
    volatile int never = 0;
    if (cta == 1) mbar_wait(bar(b_fin), 0, &never, nullptr, 100000000ull);
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Joins the pieces of requests cut at range boundaries: o = sum_i 2^(lse_i - lse) o_i.  One block per
// (request, query row), a thread per four dims, up to eight pieces' loads in flight.  Requests inside
// one range are final already.  Where a wait of the call gave up nothing is: all its outputs become NaN.
__global__ void __launch_bounds__(192) tree_pieces_kernel(const TreeArgs a, const TreeMma m) {
  const int r = blockIdx.x, x = blockIdx.y;
  if (const int failed = *m.status) {
    const int node = x / a.heads, h = x - node * a.heads;
    const int64_t row = (int64_t)r * a.nodes + node;
    for (int e = 0; e < 4; ++e)
      store_from_float(a.o + (row * a.o_sr + (int64_t)h * a.o_sh + 4 * threadIdx.x + e) * dt_size(a.o_dtype), a.o_dtype, NAN);
    if (threadIdx.x == 0 && a.lse) store_from_float(a.lse + (row * a.lse_sr + h) * dt_size(a.lse_dtype), a.lse_dtype, NAN);
    if (threadIdx.x == 0 && r == 0 && x == 0) atomicOr(&g_tree_status, failed);
    return;
  }
  __shared__ int bnd[kMaxCtas + 1];
  const int plo = __ldg(m.prefix + r), phi = __ldg(m.prefix + r + 1);
  for (int c = threadIdx.x; c <= m.ranges; c += blockDim.x) bnd[c] = __ldg(m.bounds + c);
  __syncthreads();
  auto range_of = [&](int t) {  // the non-empty range that holds tile t
    int lo = 0, hi = m.ranges;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (bnd[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  };
  if (phi == plo) return;
  const int c0 = range_of(plo), c1 = range_of(phi - 1);
  if (c0 == c1) return;
  __shared__ float wts[kMaxCtas];
  __shared__ int64_t at[kMaxCtas];
  __shared__ int np_s;
  __shared__ float inv_s;
  const int g = x >> 7, i = x & 127;
  if (threadIdx.x < 32) {
    int np = 0;
    for (int b = c0; b <= c1; b += 32) {
      const int c = b + (int)threadIdx.x;
      const bool in = c <= c1 && bnd[c] < bnd[c + 1];  // empty ranges wrote nothing
      const unsigned bal = __ballot_sync(0xffffffffu, in);
      if (in) {
        const int k = np + __popc(bal & ((1u << threadIdx.x) - 1));
        const int slot = plo <= bnd[c] ? 2 * c : 2 * c + 1;
        at[k] = ((int64_t)slot * m.groups + g) * 128 + i;
        wts[k] = __ldg(m.part_lse + at[k]);
      }
      np += __popc(bal);
    }
    __syncwarp();
    float mx = -INFINITY;
    bool bad = false;
    for (int k = threadIdx.x; k < np; k += 32) {
      mx = fmaxf(mx, wts[k]);
      bad |= wts[k] != wts[k];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    bad = __any_sync(0xffffffffu, bad);
    float sum = 0.f;
    for (int k = threadIdx.x; k < np; k += 32) {
      const float w = wts[k] == -INFINITY ? 0.f : exp2f(wts[k] - mx);
      wts[k] = w;
      sum += w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (bad) sum = NAN;
    if (threadIdx.x == 0) {
      np_s = np;
      inv_s = sum == 0.f ? 0.f : 1.f / sum;
      const int node = x / a.heads, h = x - node * a.heads;
      if (a.lse)
        store_from_float(a.lse + (((int64_t)r * a.nodes + node) * a.lse_sr + h) * dt_size(a.lse_dtype), a.lse_dtype,
                         (mx + log2f(sum)) * kLn2);
    }
  }
  __syncthreads();
  const int np = np_s, node = x / a.heads, h = x - node * a.heads;
  const float inv = inv_s;
  uint8_t* op = a.o + (((int64_t)r * a.nodes + node) * a.o_sr + (int64_t)h * a.o_sh) * dt_size(a.o_dtype);
  const int d = 4 * threadIdx.x;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < np; k0 += 8) {
    float4 v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < np) v[e] = __ldg(reinterpret_cast<const float4*>(m.part_o + at[k0 + e] * a.rank + d));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float w = k0 + e < np ? wts[k0 + e] : 0.f;
      if (w == 0.f) continue;  // a piece without visible tokens holds nothing
      acc.x += w * v[e].x;
      acc.y += w * v[e].y;
      acc.z += w * v[e].z;
      acc.w += w * v[e].w;
    }
  }
  const float r4[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  if (a.o_dtype == 0 && m.o_vec) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(r4[0], r4[1]), hi = __floats2bfloat162_rn(r4[2], r4[3]);
    *reinterpret_cast<uint2*>(op + (int64_t)d * 2) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) store_from_float(op + (int64_t)(d + e) * dt_size(a.o_dtype), a.o_dtype, r4[e]);
  }
}

}  // namespace qmla
