// Accumulated attention weight of every cached token.
//
//   weights[r][t] = decay * weights[r][t] + sum over request r's query rows (j, h) of exp(s_jht - lse_jh)
//   s_jht = (q_jh . k_t) / rms_th * sm_scale
//
// for the tokens t before the longest of the request's row lengths.  lse is what the decode of the
// same queries returned, so nothing is normalised here: one pass over the keys, one number per
// token out.  Rows whose lse is not finite (nothing visible) add nothing.
//
// The tensor-core form is one persistent CTA per SM over 128-token tiles: S^T[128 tokens, query rows] =
// K . Q^T, so that a token is a TMEM lane and the sum over the rows stays inside a thread.  The keys cross
// HBM once (2.2 GB at 64 requests of up to 32k tokens, bf16): 386-410 us, 5.3-5.7 TB/s, 81-87% of the copy
// bandwidth; over an FP8 cache, 16 requests x 4 rows x 8192 tokens, 71 us (64 of them this kernel, its preparation
// 8), 2.1 TB/s: Q of 96 rows takes 196 KB and leaves two 16 KB slots, 32 KB in flight per SM.
//
// Precision: scores are 32-bit sums of the tensor core, which rounds towards zero at each of its steps of
// 16 (32) dims; at scores of 20 a weight is off by up to 2e-5 of itself, the sums of 64 requests by 3.5e-7 against 64
// bits.  The lse of the decode comes from the same sums, so that a row's weights add up to one per head.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <cstring>
#include <type_traits>

#include "qmla.h"
#include "qmla_decode.cuh"
#include "qmla_host.cuh"
#include "qmla_pair.cuh"
#include "qmla_qimage.cuh"

using namespace qmla;

namespace {

__device__ int g_weights_status;  // bits of every call that failed on this device (qmla_operator_status)

constexpr int kMaxDim = 2048;

struct WeightArgs {
  const uint8_t *q, *q_pe;
  int64_t q_sr, q_sh, qpe_sr, qpe_sh;  // elements
  int q_dtype;
  const uint8_t* cache;
  int64_t page_b, tok_b, num_pages;
  const int32_t* bt;
  int64_t bt_stride, bt_cols;
  int page_size;
  const int32_t* lens;  // [reqs * qrows]
  int reqs, qrows, heads, rank, qk_dim, rms_mode;
  int64_t rms_off_b;
  float sm_scale, logit_cap, decay;
  const float* k_scale;
  const float* lse;
  int64_t lse_sr;
  float* w;
  int64_t w_sr, w_cols;
};

// Tokens of request r that its rows see together, within its tables.
__device__ __forceinline__ int64_t weight_len(const WeightArgs& a, int r) {
  int L = 0;
  for (int j = 0; j < a.qrows; ++j) L = max(L, __ldg(a.lens + (int64_t)r * a.qrows + j));
  return min((int64_t)L, min(a.bt_cols * a.page_size, a.w_cols));
}

// 1 / rms from the divisor's bits (one byte per head, or two); not positive counts as 1.
template <bool FP8>
__device__ __forceinline__ float inv_rms_bits(int mode, uint32_t bits, float kscale) {
  if (FP8 && mode == QMLA_RMS_LOG8) return ex2_approx(3.0f - (float)bits * (6.0f / 255.0f));
  const float rv = (!FP8 || mode == QMLA_RMS_BF16) ? __bfloat162float(__ushort_as_bfloat16((uint16_t)bits))
                                                  : e4m3_to_f32((uint8_t)bits) * kscale;
  return rv > 0.f ? 1.f / rv : 1.f;
}

// ---------------------------------------------------------------- generic kernel
// Any page size, alignment of the rms tail and number of rows; 32-bit arithmetic on the CUDA
// cores.  A warp takes a token: its lanes hold the key row's 16-byte units, each query row is one
// dot product, the weights add up in the lane-0 register.
template <bool FP8>
__global__ void __launch_bounds__(256) weights_generic_kernel(const WeightArgs a) {
  constexpr int V = FP8 ? 16 : 8;
  constexpr int kUnits = kMaxDim / V / 32;  // units per lane
  const int r = blockIdx.y, lane = threadIdx.x & 31;
  const int64_t n = weight_len(a, r);
  const float kscale = FP8 && a.k_scale ? __ldg(a.k_scale) : 1.f;
  const int es = !FP8 || a.rms_mode == QMLA_RMS_BF16 ? 2 : 1;
  const int64_t warps = (int64_t)gridDim.x * 8;
  for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < n; t += warps) {
    const int pg = __ldg(a.bt + r * a.bt_stride + t / a.page_size);
    float sum = 0.f;
    if (pg >= 0 && pg < a.num_pages) {
      const uint8_t* kr = a.cache + (int64_t)pg * a.page_b + t % a.page_size * a.tok_b;
      float kv[kUnits][V];
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int d0 = (lane + 32 * k) * V;
        alignas(16) uint8_t raw[16];
        if (d0 < a.qk_dim) *reinterpret_cast<uint4*>(raw) = __ldg(reinterpret_cast<const uint4*>(kr + lane * 16 + 512 * k));
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x = FP8 ? e4m3_to_f32(raw[e]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(raw)[e]);
          kv[k][e] = d0 + e < a.qk_dim ? x : 0.f;  // the last unit may run into the rms tail
        }
      }
      for (int j = 0; j < a.qrows; ++j) {
        const int64_t row = (int64_t)r * a.qrows + j;
        if (t >= __ldg(a.lens + row)) continue;
        for (int h = 0; h < a.heads; ++h) {
          const float lse = __ldg(a.lse + row * a.lse_sr + h);
          if (!isfinite(lse)) continue;
          float d = 0.f;
#pragma unroll
          for (int k = 0; k < kUnits; ++k) {
            const int d0 = (lane + 32 * k) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const int c = d0 + e;
              if (c < a.qk_dim) {
                const uint8_t* qp = c < a.rank ? a.q + (row * a.q_sr + h * a.q_sh + c) * 2
                                               : a.q_pe + (row * a.qpe_sr + h * a.qpe_sh + c - a.rank) * 2;
                d += kv[k][e] * load_as_float(qp, a.q_dtype);
              }
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
          float f = kscale * a.sm_scale;
          if (a.rms_mode != QMLA_RMS_NONE) {
            const uint8_t* p = kr + a.rms_off_b + es * h;
            const uint32_t bits = es == 1 ? __ldg(p) : (uint32_t)__ldg(p) | (uint32_t)__ldg(p + 1) << 8;
            f *= inv_rms_bits<FP8>(a.rms_mode, bits, kscale);
          }
          float s = d * f;
          if (a.logit_cap > 0.f) s = a.logit_cap * tanhf(s / a.logit_cap);
          sum += exp2f((s - lse) * kLog2e);
        }
      }
    }
    if (lane == 0) {
      float* w = a.w + r * a.w_sr + t;
      *w = *w * a.decay + sum;
    }
  }
}

// ---------------------------------------------------------------- tensor-core kernel
// Pages of whole 16-token runs.  One persistent CTA per SM walks a contiguous range of the 128-token
// tiles of all requests.  Per tile S^T[128 tokens, query rows] = K_tile . Q^T on tcgen05 (M = 128, a
// token per TMEM lane), so a thread of the epilogue owns a token: it turns its S columns into
// weights one after another and adds them in a register, with no exchange between threads and one
// 4-byte store.  Warp 0 streams K by TMA boxes of up to `cps` 128-byte columns x 16 tokens (a second
// load warp made no difference), warp 1 issues the MMAs, warps 2-5 and 6-9 are two epilogues for the even
// and the odd tiles; S is double-buffered.
// Bound: HBM, the QK columns and the rms tail of every cached token, once.  The kernel holds no
// values, so what shared memory Q leaves is all K in flight.
struct WeightMmaArgs {
  const int32_t* prefix;    // [reqs + 1] tiles
  const uint8_t* img;       // [reqs][img_bytes]
  const float* meta;        // [reqs][3 np]: np pairs (score scale, log2-domain lse; +inf adds nothing), np tokens seen
  uint32_t img_bytes;
  int j0, jn;               // query rows j0 .. j0 + jn - 1 of every request in this pass; column h * jn + j
  int np;                   // columns rounded up to 16
  int terms, chunks, full_chunks;
  int run, cps, nslots;     // tokens per box, columns per slot, slots per tile
  uint32_t nk, off_q, off_meta, off_bars;
  int units, base_b, skip;  // rms tail: 16-byte units read per token, first byte, bytes to skip
  int first;                // this pass applies the decay
  int q_vec;
  int* status;
  uint32_t wait_us;         // how long a wait may last
};
struct WeightMaps {
  CUtensorMap chunk;  // (element, token in page, page), box = one 128-byte column x run tokens
  CUtensorMap wide;   // (element, token in group, column, group in page, page), box = cps columns x run
};

constexpr int kWThreads = 320;  // warp 0 loads, 1 multiplies, 2-5 and 6-9 are the epilogue groups
constexpr int kWMaxRows = 128;
constexpr int kWMaxUnits = 7;  // 96 bytes of divisors (48 heads x 2) plus the misalignment

// Images of the queries, what the epilogue needs of each, and the tile prefix.  A warp per image row.
template <bool FP8>
__global__ void __launch_bounds__(256) weights_prep_kernel(const WeightArgs a, const WeightMmaArgs m, uint8_t* img,
                                                           float* meta, int32_t* prefix) {
  const int r = blockIdx.x, lane = threadIdx.x & 31;
  const int col = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int h = col / m.jn, j = m.j0 + col % m.jn;
  const bool live = h < a.heads;
  const int64_t row = (int64_t)r * a.qrows + j;
  const QSource s{a.q, a.q_pe, a.q_sr, a.q_sh, a.qpe_sr, a.qpe_sh, a.q_dtype, a.rank, a.qk_dim, m.q_vec};
  const float inv = write_q_row<FP8>(s, live ? row : -1, h, img + (int64_t)r * m.img_bytes, col, m.np, m.chunks, m.terms);
  if (lane == 0) {
    float* mt = meta + (int64_t)r * 3 * m.np;
    const float lse = live ? __ldg(a.lse + row * a.lse_sr + h) : INFINITY;
    mt[2 * col] = inv * a.sm_scale * (FP8 && a.k_scale ? __ldg(a.k_scale) : 1.f);
    mt[2 * col + 1] = isfinite(lse) ? lse * kLog2e : INFINITY;
    mt[2 * m.np + col] = __int_as_float(live ? __ldg(a.lens + row) : INT32_MAX);
  }
  if (blockIdx.x == 0 && blockIdx.y == 0) {  // exclusive prefix of the requests' tiles
    __shared__ int warp_sum[8];
    __shared__ int carry;
    if (threadIdx.x == 0) {
      carry = 0;
      prefix[0] = 0;
      *m.status = 0;
    }
    for (int base = 0; base < a.reqs; base += 256) {
      const int i = base + threadIdx.x;
      int x = i < a.reqs ? (int)((weight_len(a, i) + kTile - 1) / kTile) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) warp_sum[threadIdx.x >> 5] = x;
      __syncthreads();
      x += carry;
      for (int w = 0; w < (int)(threadIdx.x >> 5); ++w) x += warp_sum[w];
      if (i < a.reqs) prefix[i + 1] = x;
      __syncthreads();
      if (threadIdx.x == 255) carry = x;
    }
  }
}

template <bool FP8>
__global__ void __launch_bounds__(kWThreads, 1)
    weights_mma_kernel(const __grid_constant__ WeightMaps maps, const WeightArgs a, const WeightMmaArgs m) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total = __ldg(m.prefix + a.reqs);
  const int lo = (int)((int64_t)total * blockIdx.x / gridDim.x), hi = (int)((int64_t)total * (blockIdx.x + 1) / gridDim.x);
  if (lo >= hi) return;  // uniform for the CTA
  const int req0 = first_row_at(m.prefix, a.reqs, lo);
  const uint32_t slot_bytes = 16384u * m.cps;
  const uint32_t qbuf = sbase + m.off_q;
  float* meta_s = reinterpret_cast<float*>(smem + m.off_meta);  // [3][np] of the current request
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + m.off_bars);
  const uint32_t b_kfull = 0, b_kempty = m.nk, b_sfull = 2 * m.nk, b_sempty = b_sfull + 2, b_qfull = b_sempty + 2,
                 b_qempty = b_qfull + 1, b_fin = b_qempty + 1, n_bars = b_fin + 1;
  auto bar = [&](uint32_t i) { return smem_u32(bars + i); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + n_bars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + n_bars) + 1;
  const uint32_t want = 2 * m.np;
  const uint32_t tmem_cols = want <= 32 ? 32 : want <= 64 ? 64 : want <= 128 ? 128 : 256;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < m.nk; ++i) {
      mbar_init(bar(b_kfull + i), 1);
      mbar_init(bar(b_kempty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(b_sfull + i), 1);
      mbar_init(bar(b_sempty + i), 4);
    }
    mbar_init(bar(b_qfull), 1);
    mbar_init(bar(b_qempty), 1);
    mbar_init(bar(b_fin), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    // ---------------- K boxes, and each request's Q image
    const uint64_t pol = policy_evict_normal();
    const int nrun = kTile / m.run, estep = FP8 ? 128 : 64;
    SegCursor cur{req0, lo, hi};
    int r, k0, k1, plo, phi;
    uint32_t seg = 0, armed = 0;
    Ring ring;
    bool ok = true;
    while (ok && next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
      if (lane == 0) {
        if (seg > 0) ok = mbar_wait_for(bar(b_qempty), (seg - 1) & 1, abort_flag, m.status, m.wait_us);
        if (ok) {
          mbar_expect_tx(bar(b_qfull), m.img_bytes);
          load_image(qbuf, m.img + (int64_t)r * m.img_bytes, m.img_bytes, bar(b_qfull), policy_evict_last());
          ++seg;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      const int64_t n = weight_len(a, r);
      const int32_t* bt = a.bt + r * a.bt_stride;
      for (int k = k0; k < k1 && ok; ++k) {
        // page of the tile's token run `lane` (-1 past the end: zeros)
        const int64_t tok = (int64_t)k * kTile + lane * m.run;
        const int pg = lane < nrun && tok < n ? __ldg(bt + tok / a.page_size) : -1;
        const int b = lane % nrun, c = lane / nrun;
        const int mypg = __shfl_sync(0xffffffffu, pg, b);
        const int y = (int)(((int64_t)k * kTile + b * m.run) % a.page_size);
        for (int s = 0; s < m.nslots && ok; ++s) {
          const int c0 = s * m.cps, nch = min(m.cps, m.chunks - c0);
          const bool plain = c0 + m.cps > m.full_chunks;
          ok = mbar_wait_for(bar(b_kempty + ring.idx), ring.ph ^ 1, abort_flag, m.status, m.wait_us);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(bar(b_kfull + ring.idx), (uint32_t)nch * 16384u);
          const uint32_t slot = sbase + ring.idx * slot_bytes;
          if (plain) {
            if (c < nch)
              tma_load_3d(slot + c * 16384 + b * m.run * 128, &maps.chunk, (c0 + c) * estep, y, mypg,
                          bar(b_kfull + ring.idx), pol);
          } else if (lane < nrun) {
            tma_load_5d(slot + lane * m.run * m.cps * 128, &maps.wide, 0, 0, c0, y / 8, mypg, bar(b_kfull + ring.idx), pol);
          }
          ++armed;
          ring.next(m.nk);
        }
      }
    }
    if (!ok && lane == 0) {  // after an abort: wait (bounded) for the copies already issued
      volatile int never = 0;
      for (uint32_t p = armed > m.nk ? armed - m.nk : 0u; p < armed; ++p)
        mbar_wait(bar(b_kfull + p % m.nk), (p / m.nk) & 1, &never, nullptr, 20000000ull);
      if (seg > 0) mbar_wait(bar(b_qfull), (seg - 1) & 1, &never, nullptr, 20000000ull);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- S^T = K . Q^T, the whole warp issuing (qmla_pair.cuh)
    const uint32_t q_lo = sdesc_lo(qbuf, 16);
    const uint32_t qc16 = (uint32_t)m.np * 128 >> 4, qt16 = (uint32_t)(m.chunks * m.np) * 128 >> 4;
    // formats: bf16 both; or e4m3 keys and the term's format for Q
    const uint32_t idesc0 = make_idesc_f16(FP8 ? 0 : 1, 128, m.np, 0, 0);
    SegCursor cur{req0, lo, hi};
    int r, k0, k1, plo, phi;
    uint32_t jt = 0, seg = 0;
    Ring ring;
    bool ok = true;
    auto wait = [&](uint32_t b, uint32_t ph) {
      ok = ok && mbar_wait_for(bar(b), ph, abort_flag, m.status, m.wait_us);
      ok = __all_sync(0xffffffffu, ok);
    };
    while (ok && next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
      wait(b_qfull, seg & 1);
      for (int k = k0; k < k1 && ok; ++k, ++jt) {
        const uint32_t sb = jt & 1;
        if (jt >= 2) wait(b_sempty + sb, ((jt - 2) >> 1) & 1);
        tc_fence_after();
        const uint32_t d = tmem + sb * m.np;
        for (int s = 0; s < m.nslots; ++s) {
          wait(b_kfull + ring.idx, ring.ph);
          if (!ok) break;
          tc_fence_after();
          const int c0 = s * m.cps, nch = min(m.cps, m.chunks - c0);
          // column ci: plain slots keep its 128 rows together, wide ones every 8 rows
          const bool plain = c0 + m.cps > m.full_chunks;
          const uint32_t a0 = sdesc_lo(sbase + ring.idx * slot_bytes, 16), a_hi = plain ? sdesc_hi(1024) : sdesc_hi(1024 * m.cps);
          const uint32_t a_col = plain ? 16384 >> 4 : 1024 >> 4;
          for (int ci = 0; ci < nch; ++ci) {
            for (int t = 0; t < m.terms; ++t) {
              const uint32_t al = a0 + ci * a_col, bl = q_lo + (uint32_t)(c0 + ci) * qc16 + (uint32_t)t * qt16;
              const uint32_t idesc = idesc0 | (FP8 ? q_term_format(t) << 10 : 0u);
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                tc_mma_warp<FP8>(d, al + ks * 2, a_hi, bl + ks * 2, sdesc_hi(1024), idesc, ks > 0 ? 1u : (uint32_t)(s | ci | t));
            }
          }
          tc_commit_warp(bar(b_kempty + ring.idx));
          ring.next(m.nk);
        }
        if (ok) tc_commit_warp(bar(b_sfull + sb));
      }
      if (ok) tc_commit_warp(bar(b_qempty));
      ++seg;
    }
    volatile int never = 0;  // drain before TMEM is released
    __syncwarp();
    tc_commit_warp(bar(b_fin));
    mbar_wait(bar(b_fin), 0, &never, nullptr, 100000000ull);
    __syncwarp();
  } else {
    // ---------------- weights: a token per thread, a group of four warps per tile
    const int grp = (warp - 2) >> 2, sp = warp & 3, tt = sp * 32 + lane;
    const int et = threadIdx.x - 64;  // 0..255
    const float kscale = FP8 && a.k_scale ? __ldg(a.k_scale) : 1.f;
    const int es = !FP8 || a.rms_mode == QMLA_RMS_BF16 ? 2 : 1;
    const bool cap = a.logit_cap > 0.f;
    const float2* meta2 = reinterpret_cast<const float2*>(meta_s);
    const float* lim_s = meta_s + 2 * m.np;
    SegCursor cur{req0, lo, hi};
    int r, k0, k1, plo, phi;
    uint32_t jt = 0;
    bool ok = true;  // a warp that gives up still takes the barriers of the segments left
    while (next_segment(m.prefix, cur, r, k0, k1, plo, phi)) {
      named_bar_sync(1, 256);  // the previous request's meta is no longer read
      for (int i = et; i < 3 * m.np; i += 256) meta_s[i] = __ldg(m.meta + (int64_t)r * 3 * m.np + i);
      named_bar_sync(1, 256);
      const int64_t n = weight_len(a, r);
      int shortest = INT32_MAX;  // tokens that every row sees
      for (int c = lane; c < m.np; c += 32) shortest = min(shortest, __float_as_int(lim_s[c]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) shortest = min(shortest, __shfl_xor_sync(0xffffffffu, shortest, o));
      for (int k = k0; k < k1 && ok; ++k, ++jt) {
        if ((int)(jt & 1) != grp) continue;
        const int64_t t = (int64_t)k * kTile + tt;
        // this token's divisors, on their way while the tile's S is computed
        alignas(16) uint8_t tail[16 * kWMaxUnits];
        bool here = false;
        if (t < n) {
          const int pg = __ldg(a.bt + r * a.bt_stride + t / a.page_size);
          here = pg >= 0 && pg < a.num_pages;
          if (here) {
            const uint8_t* p = a.cache + (int64_t)pg * a.page_b + t % a.page_size * a.tok_b + m.base_b;
            for (int u = 0; u < m.units; ++u)
              reinterpret_cast<uint4*>(tail)[u] = __ldg(reinterpret_cast<const uint4*>(p) + u);
          }
        }
        float* wp = a.w + r * a.w_sr + t;
        const float old = t < n ? *wp : 0.f;
        ok = mbar_wait_for(bar(b_sfull + grp), (jt >> 1) & 1, abort_flag, m.status, m.wait_us);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        auto factor = [&](int h) -> float {  // of head h (0 past the last)
          if (h >= a.heads) return 0.f;
          if (m.units == 0 || !here) return 1.f;
          const uint8_t* b = tail + m.skip + es * h;
          return inv_rms_bits<FP8>(a.rms_mode, es == 1 ? *b : (uint32_t)b[0] | (uint32_t)b[1] << 8, kscale);
        };
        const uint32_t ta = tmem + ((uint32_t)(sp * 32) << 16) + grp * m.np;
        float s4[4] = {0.f, 0.f, 0.f, 0.f};
        const bool all_seen = (int64_t)(k + 1) * kTile <= shortest && !cap;
        // 16 columns at a time; column h * jn + j.  A column that adds nothing (no finite lse, or past the
        // last row) is left out by selection: its score may be NaN, or infinite like its lse.
        auto columns = [&](auto jn_c) {
          constexpr int JN = decltype(jn_c)::value;
          for (int c0 = 0; c0 < m.np; c0 += 16) {
            float x[16], f = 0.f;
            tmem_ld16(ta + c0, x);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (i % JN == 0) f = factor(c0 / JN + i / JN);
              const float2 mt = meta2[c0 + i];
              const float e = ex2_approx(x[i] * f * mt.x * kLog2e - mt.y);
              s4[i & 3] += mt.y < INFINITY ? e : 0.f;
            }
          }
        };
        if (all_seen && m.jn == 1) {
          columns(std::integral_constant<int, 1>());
        } else if (all_seen && m.jn == 2) {
          columns(std::integral_constant<int, 2>());
        } else if (all_seen && m.jn == 4) {
          columns(std::integral_constant<int, 4>());
        } else {
          float f = 0.f;
          int h = 0, j = 0;
          for (int c0 = 0; c0 < m.np; c0 += 16) {
            float x[16];
            tmem_ld16(ta + c0, x);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (j == 0) f = factor(h);
              const float2 mt = meta2[c0 + i];
              float s = x[i] * f * mt.x;
              if (cap) s = a.logit_cap * tanhf(s / a.logit_cap);
              const float e = ex2_approx(s * kLog2e - mt.y);
              if (t < __float_as_int(lim_s[c0 + i]) && mt.y < INFINITY) s4[i & 3] += e;
              if (++j == m.jn) {
                j = 0;
                ++h;
              }
            }
          }
        }
        const float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(b_sempty + grp));
        if (t < n) *wp = (m.first ? old * a.decay : old) + (here ? sum : 0.f);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicOr(&g_weights_status, QMLA_DEV_ERR_TIMEOUT);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

int check_params(const qmla_weights_params* p) {
  if (!p || p->num_reqs < 0 || p->qrows <= 0 || p->num_heads <= 0 || p->rank <= 0 || p->qk_dim < p->rank ||
      p->page_size <= 0 || p->kv_num_pages < 0 || p->block_table_cols < 0 || p->weights_cols < 0)
    return QMLA_E_INVALID;
  if (p->qk_dim > kMaxDim) return QMLA_E_UNSUPPORTED;
  if (p->q_dtype != QMLA_DT_BF16 && p->q_dtype != QMLA_DT_F16) return QMLA_E_UNSUPPORTED;
  const bool fp8 = p->kv_dtype == QMLA_DT_FP8E4M3;
  if (!fp8 && p->kv_dtype != QMLA_DT_BF16) return QMLA_E_UNSUPPORTED;
  if (p->rms_mode < 0 || p->rms_mode > 3 || (!fp8 && p->rms_mode >= 2)) return QMLA_E_INVALID;
  const int es = fp8 ? 1 : 2;
  if (reinterpret_cast<uintptr_t>(p->kv_cache) % 16 != 0 || p->kv_stride_token * es % 16 != 0 ||
      p->kv_stride_page * es % 16 != 0)
    return QMLA_E_ALIGNMENT;
  if (p->kv_row_width < p->qk_dim || p->kv_stride_token < p->kv_row_width) return QMLA_E_INVALID;
  if (p->rms_mode != QMLA_RMS_NONE) {
    const int64_t tail = (int64_t)p->num_heads * (fp8 && p->rms_mode == QMLA_RMS_BF16 ? 2 : 1);
    if (p->rms_offset < p->qk_dim || p->rms_offset + tail > p->kv_row_width) return QMLA_E_INVALID;
  }
  if ((int64_t)p->num_reqs * p->qrows > INT32_MAX || p->num_reqs > 65535) return QMLA_E_UNSUPPORTED;
  return QMLA_OK;
}

struct WeightPlan {
  bool mma;
  WeightMmaArgs m;
  int jn;  // query rows of a request in one pass of the tensor-core kernel
  uint32_t smem;
  int64_t ws_status, ws_prefix, ws_meta, ws_img, ws_total;
};

// The tensor-core kernel takes pages of whole 16-token runs, a QK width of at least two 128-byte
// columns, divisors within whole 16-byte units of the row, and as many of a request's query rows per
// pass as fit beside two K slots (96 rows of 1000 dims); further rows take further passes over the keys.
void plan_mma(const qmla_weights_params* p, const DevInfo& di, WeightPlan* pl) {
  pl->mma = false;
  pl->ws_total = 0;
  const bool fp8 = p->kv_dtype == QMLA_DT_FP8E4M3;
  const int es = fp8 ? 1 : 2;
  WeightMmaArgs& m = pl->m;
  memset(&m, 0, sizeof(m));
  m.run = gcd_int(p->page_size, kTile);
  m.chunks = (p->qk_dim * es + 127) / 128;
  m.full_chunks = p->qk_dim * es / 128;
  m.terms = q_terms(fp8, p->q_dtype);
  if (m.run < 16 || m.full_chunks < 2) return;
  if (p->rms_mode != QMLA_RMS_NONE) {
    const int bytes = p->num_heads * (!fp8 || p->rms_mode == QMLA_RMS_BF16 ? 2 : 1);
    const int off = p->rms_offset * es;
    m.base_b = off & ~15;
    m.skip = off - m.base_b;
    m.units = (m.skip + bytes + 15) / 16;
    if (m.units > kWMaxUnits || m.base_b + 16 * m.units > p->kv_row_width * es) return;
  }
  const int most = std::min(di.max_smem, kMaxDynSmem) - 1024;
  for (int jn = p->qrows; jn >= 1; --jn) {
    const int np = (jn * p->num_heads + 15) / 16 * 16;
    if (np > kWMaxRows) continue;
    const int64_t q = (int64_t)m.terms * m.chunks * np * 128;
    const int meta = 12 * np, bars = 8 * (2 * 8 + 7) + 16;  // 8 slots at most
    const int64_t ring = most - q - meta - bars;
    if (ring < 2 * 16384) continue;
    m.cps = ring >= 3 * 32768 ? 2 : 1;
    m.nk = (uint32_t)std::min<int64_t>(8, ring / (16384 * m.cps));
    m.nslots = (m.chunks + m.cps - 1) / m.cps;
    m.np = np;
    m.img_bytes = (uint32_t)q;
    m.off_q = m.nk * 16384u * m.cps;
    m.off_meta = m.off_q + (uint32_t)q;
    m.off_bars = m.off_meta + meta;
    pl->smem = m.off_bars + bars + 1024;
    pl->jn = jn;
    pl->mma = true;
    break;
  }
  if (!pl->mma) return;
  int64_t w = 0;
  pl->ws_status = w;
  w += 256;
  pl->ws_prefix = w;
  w = align_up(w + 4 * ((int64_t)p->num_reqs + 1), 256);
  pl->ws_meta = w;
  w = align_up(w + (int64_t)12 * m.np * p->num_reqs, 256);
  pl->ws_img = w;
  w = align_up(w + (int64_t)m.img_bytes * p->num_reqs, 256);
  pl->ws_total = w;
}

template <bool FP8>
int launch_mma(const qmla_weights_params* p, const WeightArgs& a, const WeightPlan& pl, const DevInfo& di, uint8_t* ws,
               cudaStream_t st) {
  const int es = FP8 ? 1 : 2;
  WeightMmaArgs m = pl.m;
  m.status = reinterpret_cast<int*>(ws + pl.ws_status);
  m.wait_us = wait_limit_us();
  m.prefix = reinterpret_cast<const int32_t*>(ws + pl.ws_prefix);
  m.meta = reinterpret_cast<const float*>(ws + pl.ws_meta);
  m.img = ws + pl.ws_img;
  m.q_vec = q_vec(a.q, a.q_sr, a.q_sh, a.q_pe, a.qpe_sr, a.qpe_sh, a.rank, a.qk_dim);
  WeightMaps maps;
  const cuuint64_t tok = p->kv_stride_token * es, page = p->kv_stride_page * es;
  const cuuint32_t col = 128 / es;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)p->qk_dim, (cuuint64_t)p->page_size, (cuuint64_t)p->kv_num_pages};
    const cuuint64_t strides[2] = {tok, page};
    const cuuint32_t box[3] = {col, (cuuint32_t)m.run, 1};
    if (!encode_tiled(&maps.chunk, FP8, p->kv_cache, 3, dims, strides, box)) return QMLA_E_ALIGNMENT;
  }
  {
    const cuuint64_t dims[5] = {col, 8, (cuuint64_t)m.full_chunks, (cuuint64_t)(p->page_size / 8), (cuuint64_t)p->kv_num_pages};
    const cuuint64_t strides[4] = {tok, 128, 8 * tok, page};
    const cuuint32_t box[5] = {col, 8, (cuuint32_t)m.cps, (cuuint32_t)(m.run / 8), 1};
    if (!encode_tiled(&maps.wide, FP8, p->kv_cache, 5, dims, strides, box)) return QMLA_E_ALIGNMENT;
  }
  if (!allow_smem(weights_mma_kernel<FP8>, kMaxDynSmem)) return QMLA_E_CUDA;
  for (int j0 = 0; j0 < a.qrows; j0 += pl.jn) {
    m.j0 = j0;
    m.jn = std::min(pl.jn, a.qrows - j0);
    m.first = j0 == 0;
    weights_prep_kernel<FP8><<<dim3(a.reqs, m.np / 8), 256, 0, st>>>(a, m, ws + pl.ws_img,
                                                                     reinterpret_cast<float*>(ws + pl.ws_meta),
                                                                     reinterpret_cast<int32_t*>(ws + pl.ws_prefix));
    weights_mma_kernel<FP8><<<di.sms, kWThreads, pl.smem, st>>>(maps, a, m);
  }
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
}

}  // namespace

int qmla::weights_status(bool clear, cudaStream_t st, int32_t* bits) { return take_status(&g_weights_status, clear, st, bits); }

extern "C" {

int qmla_weights_workspace_bytes(const qmla_weights_params* p, int64_t* bytes) try {
  if (!bytes) return QMLA_E_INVALID;
  const int rc = check_params(p);
  if (rc != QMLA_OK) return rc;
  const DevInfo di = dev_info(p->device);
  if (!di.ok) return QMLA_E_CUDA;
  WeightPlan pl;
  plan_mma(p, di, &pl);
  *bytes = pl.ws_total;
  return QMLA_OK;
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

int qmla_accumulate_weights(const qmla_weights_params* p, void* stream) try {
  int rc = check_params(p);
  if (rc != QMLA_OK) return rc;
  if (p->num_reqs == 0) return QMLA_OK;
  if (!p->q || (!p->q_pe && p->qk_dim > p->rank) || !p->kv_cache || !p->block_table || !p->seq_lens || !p->lse ||
      !p->weights)
    return QMLA_E_INVALID;
  const DevInfo di = dev_info(p->device);
  if (!di.ok) return QMLA_E_CUDA;
  DeviceGuard dg(p->device);
  if (!dg.ok()) return QMLA_E_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool fp8 = p->kv_dtype == QMLA_DT_FP8E4M3;
  const int es = fp8 ? 1 : 2;
  WeightArgs a;
  memset(&a, 0, sizeof(a));
  a.q = reinterpret_cast<const uint8_t*>(p->q);
  a.q_pe = reinterpret_cast<const uint8_t*>(p->q_pe ? p->q_pe : p->q);
  a.q_sr = p->q_stride_row;
  a.q_sh = p->q_stride_head;
  a.qpe_sr = p->qpe_stride_row;
  a.qpe_sh = p->qpe_stride_head;
  a.q_dtype = p->q_dtype;
  a.cache = reinterpret_cast<const uint8_t*>(p->kv_cache);
  a.page_b = p->kv_stride_page * es;
  a.tok_b = p->kv_stride_token * es;
  a.num_pages = p->kv_num_pages;
  a.bt = p->block_table;
  a.bt_stride = p->block_table_stride;
  a.bt_cols = p->block_table_cols;
  a.page_size = p->page_size;
  a.lens = p->seq_lens;
  a.reqs = p->num_reqs;
  a.qrows = p->qrows;
  a.heads = p->num_heads;
  a.rank = p->rank;
  a.qk_dim = p->qk_dim;
  a.rms_mode = p->rms_mode;
  a.rms_off_b = (int64_t)p->rms_offset * es;
  a.sm_scale = p->sm_scale;
  a.logit_cap = p->logit_cap;
  a.decay = p->decay;
  a.k_scale = p->k_scale;
  a.lse = p->lse;
  a.lse_sr = p->lse_stride_row;
  a.w = p->weights;
  a.w_sr = p->weights_stride_req;
  a.w_cols = p->weights_cols;
  WeightPlan pl;
  plan_mma(p, di, &pl);
  if (pl.mma) {
    if (!p->workspace || p->workspace_bytes < pl.ws_total) return QMLA_E_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0) return QMLA_E_ALIGNMENT;
    uint8_t* ws = reinterpret_cast<uint8_t*>(p->workspace);
    return fp8 ? launch_mma<true>(p, a, pl, di, ws, st) : launch_mma<false>(p, a, pl, di, ws, st);
  }
  const dim3 grid((unsigned)std::max(1, 8 * di.sms / p->num_reqs), p->num_reqs);
  if (fp8)
    weights_generic_kernel<true><<<grid, 256, 0, st>>>(a);
  else
    weights_generic_kernel<false><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

}  // extern "C"
