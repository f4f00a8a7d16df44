// Attention of a drafted token tree over the paged latent cache.
//
// Request r has ctx committed tokens and T drafted ones whose rows sit behind them in its pages.
// Node i sees tokens [0, ctx) and the drafted tokens of its 64-bit mask (itself and its
// ancestors):  s = (q . k) / rms(token, head) * sm_scale,  o = softmax(s) . latent,
// lse = ln sum exp s.  A node with an empty mask is padding: o = 0, lse = -inf.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstring>
#include <map>
#include <mutex>

#include "qmla.h"
#include "qmla_decode.cuh"
#include "qmla_host.cuh"
#include "qmla_tree_mma.cuh"

using namespace qmla;

namespace {

constexpr int kGenThreads = 256;
constexpr int kGenTile = 32;   // tokens per step of the generic kernel
constexpr int kGenHeads = 8;   // heads per block of the generic kernel, one softmax warp each
constexpr int kMaxNodes = 64;
constexpr int kMaxRank = 2048;

// 1 / rms(token, head) of a cache row; a divisor that is not positive counts as 1.
template <bool FP8>
__device__ __forceinline__ float inv_rms(const TreeArgs& a, const uint8_t* row, int h, float kscale) {
  if (a.rms_mode == QMLA_RMS_NONE) return 1.f;
  const uint8_t* p = row + a.rms_off_b;
  if (FP8 && a.rms_mode == QMLA_RMS_LOG8) return ex2_approx(3.0f - (float)__ldg(p + h) * (6.0f / 255.0f));
  float rv;
  if (!FP8)
    rv = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[h]);
  else if (a.rms_mode == QMLA_RMS_BF16)  // raw bytes: the offset may be odd
    rv = __bfloat162float(__ushort_as_bfloat16((uint16_t)(__ldg(p + 2 * h) | (__ldg(p + 2 * h + 1) << 8))));
  else
    rv = e4m3_to_f32(__ldg(p + h)) * kscale;
  return rv > 0.f ? 1.f / rv : 1.f;
}

// ---------------------------------------------------------------- generic kernel
// Any rank, page size and head count; 32-bit arithmetic on the CUDA cores.  One block per
// (node, 8 heads, split of the tokens).  Per 32-token step: each warp scores 4 tokens against the
// 8 heads (a lane takes a 16-byte unit of the key row), then warp h updates head h's running
// maximum and sum, then every thread adds the visible tokens' values to its output dims.  Values of
// tokens that the node does not see are not read, so what they hold cannot matter.
template <bool FP8>
__global__ void __launch_bounds__(kGenThreads) tree_generic_kernel(const TreeArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int V = FP8 ? 16 : 8;  // elements per 16-byte unit
  const int units = (a.qk_dim + V - 1) / V;
  float* qs = reinterpret_cast<float*>(smem);  // [8][units * V], zero past qk_dim
  const int qst = units * V;
  __shared__ float s_s[kGenTile][kGenHeads];
  __shared__ float p_s[kGenTile][kGenHeads];
  __shared__ float alpha_s[kGenHeads], l_s[kGenHeads];
  __shared__ const uint8_t* rows_s[kGenTile];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hgroups = (a.heads + kGenHeads - 1) / kGenHeads;
  const int row = blockIdx.x / hgroups, h0 = (blockIdx.x - row * hgroups) * kGenHeads;
  const int nh = min(kGenHeads, a.heads - h0);
  const int r = row / a.nodes, node = row - r * a.nodes;
  const float kscale = FP8 && a.k_scale ? __ldg(a.k_scale) : 1.f;
  const uint64_t mask = (uint64_t)__ldg(reinterpret_cast<const long long*>(a.mask) + r * a.mask_stride + node);
  const int ctx = tree_ctx(a, r);
  // tokens this node may see: up to its last visible draft
  int64_t n = mask ? (int64_t)ctx + 64 - __clzll((long long)mask) : 0;
  n = min(n, min(a.bt_cols * a.page_size, (int64_t)ctx + a.nodes));
  const int64_t tiles = (n + kGenTile - 1) / kGenTile;
  const int64_t t_lo = tiles * blockIdx.y / a.nsplit, t_hi = tiles * (blockIdx.y + 1) / a.nsplit;
  for (int i = tid; i < kGenHeads * qst; i += kGenThreads) {
    const int h = i / qst, d = i - h * qst;
    float v = 0.f;
    if (h < nh && d < a.qk_dim) {
      const uint8_t* src = d < a.rank ? a.q + ((int64_t)row * a.q_sr + (int64_t)(h0 + h) * a.q_sh + d) * 2
                                      : a.q_pe + ((int64_t)row * a.qpe_sr + (int64_t)(h0 + h) * a.qpe_sh + d - a.rank) * 2;
      v = load_as_float(src, a.q_dtype);
    }
    qs[i] = v;
  }
  float acc[kMaxRank / kGenThreads][kGenHeads];
#pragma unroll
  for (int k = 0; k < kMaxRank / kGenThreads; ++k)
#pragma unroll
    for (int h = 0; h < kGenHeads; ++h) acc[k][h] = 0.f;
  float m = -INFINITY, l = 0.f;  // warp h: head h0 + h
  __syncthreads();
  for (int64_t t = t_lo; t < t_hi; ++t) {
    const int64_t tok0 = t * kGenTile;
    for (int j = warp; j < kGenTile; j += kGenThreads / 32) {
      const int64_t tok = tok0 + j;
      bool see = tok < n;
      if (see && tok >= ctx) see = mask >> (tok - ctx) & 1;
      const uint8_t* kr = nullptr;
      if (see) {
        const int pg = __ldg(a.bt + r * a.bt_stride + tok / a.page_size);
        if (pg >= 0 && pg < a.num_pages)
          kr = a.cache + (int64_t)pg * a.page_b + tok % a.page_size * a.tok_b;
        see = kr != nullptr;  // a page id outside the cache: the token counts as absent
      }
      float d[kGenHeads];
#pragma unroll
      for (int h = 0; h < kGenHeads; ++h) d[h] = 0.f;
      if (see) {
        for (int u = lane; u < units; u += 32) {
          alignas(16) uint8_t raw[16];
          *reinterpret_cast<uint4*>(raw) = __ldg(reinterpret_cast<const uint4*>(kr) + u);
          float kv[V];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float x = FP8 ? e4m3_to_f32(raw[e]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(raw)[e]);
            kv[e] = u * V + e < a.qk_dim ? x : 0.f;  // the unit may run into the rms tail
          }
#pragma unroll
          for (int h = 0; h < kGenHeads; ++h) {
            const float4* q4 = reinterpret_cast<const float4*>(qs + h * qst + u * V);
#pragma unroll
            for (int e = 0; e < V / 4; ++e) {
              const float4 qv = q4[e];
              d[h] += qv.x * kv[4 * e] + qv.y * kv[4 * e + 1] + qv.z * kv[4 * e + 2] + qv.w * kv[4 * e + 3];
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < kGenHeads; ++h)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d[h] += __shfl_xor_sync(0xffffffffu, d[h], o);
      if (lane < kGenHeads) {
        float x = -INFINITY;
        if (see && lane < nh) {
          float dh = d[0];
#pragma unroll
          for (int h = 1; h < kGenHeads; ++h) dh = lane == h ? d[h] : dh;
          x = dh * kscale * inv_rms<FP8>(a, kr, h0 + lane, kscale) * a.sm_scale;
          if (a.logit_cap > 0.f) x = a.logit_cap * tanhf(x / a.logit_cap);
          x *= kLog2e;
        }
        s_s[j][lane] = x;
      }
      if (lane == 0) rows_s[j] = see ? kr : nullptr;
    }
    __syncthreads();
    {
      const float x = s_s[lane][warp];
      float mx = x;
      bool bad = x != x;  // fmaxf drops a NaN: carry it into the sum instead
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m, mx);
      const float al = m == mn ? 1.f : exp2f(m - mn);
      float p = bad ? x : (x == -INFINITY ? 0.f : exp2f(x - mn));
      p_s[lane][warp] = p;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) p += __shfl_xor_sync(0xffffffffu, p, o);
      l = l * al + p;
      m = mn;
      if (lane == 0) alpha_s[warp] = al;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMaxRank / kGenThreads; ++k) {
      const int dcol = tid + k * kGenThreads;
      if (dcol < a.rank) {
#pragma unroll
        for (int h = 0; h < kGenHeads; ++h) acc[k][h] *= alpha_s[h];
        for (int j = 0; j < kGenTile; ++j) {
          const uint8_t* kr = rows_s[j];
          if (!kr) continue;
          const float v = FP8 ? e4m3_to_f32(__ldg(kr + dcol)) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(kr)[dcol]);
#pragma unroll
          for (int h = 0; h < kGenHeads; ++h) acc[k][h] += p_s[j][h] * v;
        }
      }
    }
    __syncthreads();
  }
  if (lane == 0) {
    alpha_s[warp] = m;
    l_s[warp] = l;
  }
  __syncthreads();
  const int64_t prow = ((int64_t)blockIdx.y * a.reqs * a.nodes + row) * a.heads + h0;
  for (int h = 0; h < nh; ++h) {
    const float lt = l_s[h];
    const float inv = lt == 0.f ? 0.f : kscale / lt;
#pragma unroll
    for (int k = 0; k < kMaxRank / kGenThreads; ++k) {
      const int dcol = tid + k * kGenThreads;
      if (dcol >= a.rank) continue;
      float v = acc[k][0];
#pragma unroll
      for (int g = 1; g < kGenHeads; ++g) v = g == h ? acc[k][g] : v;
      v *= inv;
      if (a.nsplit == 1)
        store_from_float(a.o + ((int64_t)row * a.o_sr + (int64_t)(h0 + h) * a.o_sh + dcol) * dt_size(a.o_dtype), a.o_dtype, v);
      else
        a.part_o[(prow + h) * a.rank + dcol] = v;
    }
  }
  if (tid < nh) {
    const float l2 = alpha_s[tid] + log2f(l_s[tid]);  // -inf where nothing is visible
    if (a.nsplit > 1)
      a.part_lse[prow + tid] = l2;
    else if (a.lse)
      store_from_float(a.lse + ((int64_t)row * a.lse_sr + h0 + tid) * dt_size(a.lse_dtype), a.lse_dtype, l2 * kLn2);
  }
}

// Joins the splits of a (row, head): o = sum_i 2^(lse_i - lse) o_i.  Splits without tokens carry
// lse = -inf and are not read; a NaN of any split is a NaN of the result.
__global__ void __launch_bounds__(128) tree_join_kernel(const TreeArgs a) {
  const int64_t rh = blockIdx.x;
  const int64_t n = (int64_t)a.reqs * a.nodes * a.heads;
  const int64_t row = rh / a.heads;
  const int h = (int)(rh - row * a.heads);
  float m = -INFINITY;
  bool bad = false;
  for (int s = 0; s < a.nsplit; ++s) {
    const float l = __ldg(a.part_lse + s * n + rh);
    m = fmaxf(m, l);
    bad |= l != l;
  }
  float sum = 0.f;
  for (int s = 0; s < a.nsplit; ++s) {
    const float l = __ldg(a.part_lse + s * n + rh);
    sum += l == -INFINITY ? 0.f : exp2f(l - m);
  }
  if (bad) sum = NAN;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint8_t* orow = a.o + (row * a.o_sr + (int64_t)h * a.o_sh) * dt_size(a.o_dtype);
  for (int d = threadIdx.x; d < a.rank; d += blockDim.x) {
    float acc = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
      const float l = __ldg(a.part_lse + s * n + rh);
      if (l != -INFINITY) acc += exp2f(l - m) * __ldg(a.part_o + (s * n + rh) * a.rank + d);
    }
    store_from_float(orow + (int64_t)d * dt_size(a.o_dtype), a.o_dtype, acc * inv);
  }
  if (threadIdx.x == 0 && a.lse)
    store_from_float(a.lse + (row * a.lse_sr + h) * dt_size(a.lse_dtype), a.lse_dtype, (m + log2f(sum)) * kLn2);
}

struct TreePlan {
  int nsplit;                     // generic kernel
  int64_t ws_lse, ws_o, ws_total;
  bool mma;                       // tensor-core kernel
  TreeMma m;
  uint32_t smem;
  int64_t ws_status, ws_prefix, ws_bounds, ws_img, ws_qinv, ws_tail;
};

// Clusters of the tensor-core kernel that can be resident at once on `device`, whatever device is current
// (asked once for each); -1 when the device cannot be asked, which is not remembered.  Lets the kernel have
// its shared memory there.
template <bool FP8, int TERMS>
int resident_clusters(int device) {
  static std::mutex mu;
  static std::map<int, int> known;
  std::lock_guard<std::mutex> lk(mu);
  auto it = known.find(device);
  if (it != known.end()) return it->second;
  DeviceGuard dg(device);
  if (!dg.ok() || !allow_smem(tree_mma_kernel<FP8, TERMS>, kMaxDynSmem)) return -1;
  int n = 0;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(kTrThreads);
  cfg.dynamicSmemBytes = kMaxDynSmem;
  if (cudaOccupancyMaxActiveClusters(&n, tree_mma_kernel<FP8, TERMS>, &cfg) != cudaSuccess) {
    cudaGetLastError();  // the error is the caller's return code, not the next launch's
    return -1;
  }
  known[device] = n;
  return n;
}

// The tensor-core kernel takes ranks of whole 128-dim columns up to 768, pages of whole 16-token runs,
// divisors within whole 16-byte units of the row, a query image and a factor table (528 bytes per head) that
// leave room for three K / V slots (not f16 queries of rank 768, nor 48 heads over an FP8 cache of that
// rank), and no more groups of 128 query rows than there are clusters.  Everything else is the
// generic kernel's.
int plan_mma(const qmla_tree_params* p, const DevInfo& di, TreePlan* pl) {
  pl->mma = false;
  const bool fp8 = p->kv_dtype == QMLA_DT_FP8E4M3;
  const int es = fp8 ? 1 : 2;
  TreeMma& m = pl->m;
  memset(&m, 0, sizeof(m));
  if (p->rank % 128 != 0 || p->rank > 768 || p->block_table_cols == 0 || p->num_reqs == 0 || p->num_nodes == 0)
    return QMLA_OK;
  m.run = gcd_int(p->page_size, 64);
  m.chunks = (p->qk_dim * es + 127) / 128;
  m.full_chunks = p->qk_dim * es / 128;
  m.v_chunks = p->rank * es / 128;
  m.terms = q_terms(fp8, p->q_dtype);
  if (m.run < 16 || m.full_chunks < 2) return QMLA_OK;
  if (p->rms_mode != QMLA_RMS_NONE) {
    const int bytes = p->num_heads * (!fp8 || p->rms_mode == QMLA_RMS_BF16 ? 2 : 1);
    const int off = p->rms_offset * es;
    m.base_b = off & ~15;
    m.skip = off - m.base_b;
    m.units = (m.skip + bytes + 15) / 16;
    if (m.units > 7 || m.base_b + 16 * m.units > p->kv_row_width * es) return QMLA_OK;
  }
  const int64_t rows = (int64_t)p->num_nodes * p->num_heads;
  const int dev = p->device;
  const int clusters = fp8 ? (m.terms == 2 ? resident_clusters<true, 2>(dev) : resident_clusters<true, 3>(dev))
                           : (m.terms == 1 ? resident_clusters<false, 1>(dev) : resident_clusters<false, 2>(dev));
  if (clusters < 0) return QMLA_E_CUDA;
  if (rows > (int64_t)128 * clusters) return QMLA_OK;
  m.rows = (int)rows;
  m.groups = (int)((rows + 127) / 128);
  m.ranges = std::min(clusters / m.groups, kMaxCtas);
  const int64_t img = (int64_t)m.terms * m.chunks * kTrRows * 128;
  const int64_t fac = (int64_t)p->num_heads * kTrFacPitch * 4;
  const int64_t ring = std::min(di.max_smem, kMaxDynSmem) - 1024 - img - tr_p_bytes(fp8) - fac - 2048;
  if (ring < 3 * (int64_t)kTrSlot) return QMLA_OK;
  m.nslots = (uint32_t)std::min<int64_t>(kTrMaxSlots, ring / kTrSlot);
  m.img_bytes = (uint32_t)img;
  m.off_q = m.nslots * kTrSlot;
  m.off_p = m.off_q + (uint32_t)img;
  m.off_fac = m.off_p + tr_p_bytes(fp8);
  m.off_misc = m.off_fac + (uint32_t)fac;
  pl->smem = m.off_misc + 2048 + 1024;
  m.seg_cost = 2;
  m.o_cols = fp8 ? (p->rank + 255) / 256 * 128 : p->rank / 2;
  int64_t w = 0;
  pl->ws_status = w;
  w += 256;
  pl->ws_prefix = w;
  w = align_up(w + 4 * ((int64_t)p->num_reqs + 1), 256);
  pl->ws_bounds = w;
  w = align_up(w + 4 * ((int64_t)m.ranges + 1), 256);
  pl->ws_img = w;
  w = align_up(w + img * 2 * m.groups * p->num_reqs, 256);
  pl->ws_qinv = w;
  w = align_up(w + (int64_t)4 * 128 * m.groups * p->num_reqs, 256);
  pl->ws_tail = w;
  w = align_up(w + (int64_t)p->num_reqs * kTrTail * p->rank * es, 256);
  pl->ws_lse = w;
  w = align_up(w + (int64_t)2 * m.ranges * m.groups * 128 * 4, 256);
  pl->ws_o = w;
  w = align_up(w + (int64_t)2 * m.ranges * m.groups * 128 * 4 * p->rank, 256);
  pl->ws_total = w;
  pl->mma = true;
  return QMLA_OK;
}

int make_tree_plan(const qmla_tree_params* p, TreePlan* pl) {
  if (!p || p->num_reqs < 0 || p->num_nodes < 0 || p->num_heads <= 0 || p->rank <= 0 || p->qk_dim < p->rank ||
      p->page_size <= 0 || p->kv_num_pages < 0 || p->block_table_cols < 0)
    return QMLA_E_INVALID;
  if (p->num_nodes > kMaxNodes || p->rank > kMaxRank || p->qk_dim > kMaxRank) return QMLA_E_UNSUPPORTED;
  if (p->q_dtype != QMLA_DT_BF16 && p->q_dtype != QMLA_DT_F16) return QMLA_E_UNSUPPORTED;
  if (p->o_dtype < 0 || p->o_dtype > 2 || p->lse_dtype < 0 || p->lse_dtype > 2) return QMLA_E_UNSUPPORTED;
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
  const DevInfo di = dev_info(p->device);
  if (!di.ok) return QMLA_E_CUDA;
  const int64_t rows = (int64_t)p->num_reqs * p->num_nodes;
  const int64_t blocks = rows * ((p->num_heads + kGenHeads - 1) / kGenHeads);
  if (blocks > INT32_MAX || rows * p->num_heads > INT32_MAX) return QMLA_E_UNSUPPORTED;
  const int rc = plan_mma(p, di, pl);
  if (rc != QMLA_OK || pl->mma) return rc;
  // tokens split over blocks until every SM has two
  pl->nsplit = blocks == 0 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(64, 2 * di.sms / blocks));
  int64_t w = 0;
  pl->ws_lse = w;
  if (pl->nsplit > 1) w = align_up(w + 4 * rows * p->num_heads * pl->nsplit, 256);
  pl->ws_o = w;
  if (pl->nsplit > 1) w = align_up(w + 4 * rows * p->num_heads * p->rank * pl->nsplit, 256);
  pl->ws_total = w;
  return QMLA_OK;
}

template <bool FP8>
int launch_generic(const TreeArgs& a, cudaStream_t st) {
  const int V = FP8 ? 16 : 8;
  const int smem = kGenHeads * ((a.qk_dim + V - 1) / V * V) * 4;
  if (!allow_smem(tree_generic_kernel<FP8>, kGenHeads * kMaxRank * 4)) return QMLA_E_CUDA;
  const int hgroups = (a.heads + kGenHeads - 1) / kGenHeads;
  tree_generic_kernel<FP8><<<dim3(a.reqs * a.nodes * hgroups, a.nsplit), kGenThreads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
}

template <bool FP8>
int launch_tree_mma(const qmla_tree_params* p, const TreeArgs& a, const TreePlan& pl, uint8_t* ws, cudaStream_t st) {
  const int es = FP8 ? 1 : 2;
  TreeMma m = pl.m;
  m.status = reinterpret_cast<int*>(ws + pl.ws_status);
  m.wait_us = wait_limit_us();
  m.prefix = reinterpret_cast<int32_t*>(ws + pl.ws_prefix);
  m.bounds = reinterpret_cast<int32_t*>(ws + pl.ws_bounds);
  m.img = ws + pl.ws_img;
  m.q_inv = reinterpret_cast<float*>(ws + pl.ws_qinv);
  m.tail = ws + pl.ws_tail;
  m.part_lse = reinterpret_cast<float*>(ws + pl.ws_lse);
  m.part_o = reinterpret_cast<float*>(ws + pl.ws_o);
  const int osz = p->o_dtype == QMLA_DT_F32 ? 4 : 2;
  m.o_vec = reinterpret_cast<uintptr_t>(p->o) % 16 == 0 && p->o_stride_row * osz % 16 == 0 && p->o_stride_head * osz % 16 == 0;
  m.q_vec = q_vec(a.q, a.q_sr, a.q_sh, a.q_pe, a.qpe_sr, a.qpe_sh, a.rank, a.qk_dim);
  TreeMaps maps;
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
    const cuuint32_t box[5] = {col, 8, 2, (cuuint32_t)(m.run / 8), 1};
    if (!encode_tiled(&maps.wide, FP8, p->kv_cache, 5, dims, strides, box)) return QMLA_E_ALIGNMENT;
  }
  {
    const cuuint64_t dims[2] = {(cuuint64_t)p->rank, (cuuint64_t)p->num_reqs * kTrTail};
    const cuuint64_t strides[1] = {(cuuint64_t)p->rank * es};
    const cuuint32_t box[2] = {col, 64};
    if (!encode_tiled(&maps.tail, FP8, m.tail, 2, dims, strides, box)) return QMLA_E_ALIGNMENT;
  }
  const int64_t warps = (int64_t)p->num_reqs * (m.groups * 128 + kTrTail);
  if (warps / 8 + 1 > INT32_MAX) return QMLA_E_UNSUPPORTED;
  tree_prep_kernel<FP8><<<(unsigned)((warps + 7) / 8 + 1), 256, 0, st>>>(a, m);
  const int grid = 2 * m.ranges * m.groups;
  constexpr int T0 = FP8 ? 2 : 1;
  if (m.terms == T0)
    tree_mma_kernel<FP8, T0><<<grid, kTrThreads, pl.smem, st>>>(maps, a, m);
  else
    tree_mma_kernel<FP8, T0 + 1><<<grid, kTrThreads, pl.smem, st>>>(maps, a, m);
  tree_pieces_kernel<<<dim3(p->num_reqs, m.rows), p->rank / 4, 0, st>>>(a, m);
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
}

}  // namespace

extern "C" {

int qmla_tree_workspace_bytes(const qmla_tree_params* p, int64_t* bytes) try {
  if (!bytes) return QMLA_E_INVALID;
  TreePlan pl;
  const int rc = make_tree_plan(p, &pl);
  if (rc != QMLA_OK) return rc;
  *bytes = pl.ws_total;
  return QMLA_OK;
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

int qmla_operator_status(int32_t device, int32_t clear, void* stream, int32_t* status) try {
  if (!status) return QMLA_E_INVALID;
  DeviceGuard dg(device);
  if (!dg.ok()) return QMLA_E_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int32_t tree = 0, weights = 0;
  if (take_status(&g_tree_status, clear != 0, st, &tree) != 0 || weights_status(clear != 0, st, &weights) != 0) return QMLA_E_CUDA;
  *status = tree | weights;
  return QMLA_OK;
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

int qmla_tree_attention(const qmla_tree_params* p, void* stream) try {
  TreePlan pl;
  int rc = make_tree_plan(p, &pl);
  if (rc != QMLA_OK) return rc;
  if (p->num_reqs == 0 || p->num_nodes == 0) return QMLA_OK;
  if (!p->q || (!p->q_pe && p->qk_dim > p->rank) || !p->kv_cache || !p->block_table || !p->ctx_lens ||
      !p->tree_mask || !p->o)
    return QMLA_E_INVALID;
  if (pl.ws_total > 0) {
    if (!p->workspace || p->workspace_bytes < pl.ws_total) return QMLA_E_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0) return QMLA_E_ALIGNMENT;
  }
  DeviceGuard dg(p->device);
  if (!dg.ok()) return QMLA_E_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool fp8 = p->kv_dtype == QMLA_DT_FP8E4M3;
  const int es = fp8 ? 1 : 2;
  uint8_t* ws = reinterpret_cast<uint8_t*>(p->workspace);
  TreeArgs a;
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
  a.ctx = p->ctx_lens;
  a.mask = p->tree_mask;
  a.mask_stride = p->mask_stride;
  a.reqs = p->num_reqs;
  a.nodes = p->num_nodes;
  a.heads = p->num_heads;
  a.rank = p->rank;
  a.qk_dim = p->qk_dim;
  a.rms_mode = p->rms_mode;
  a.rms_off_b = (int64_t)p->rms_offset * es;
  a.sm_scale = p->sm_scale;
  a.logit_cap = p->logit_cap;
  a.k_scale = p->k_scale;
  a.o = reinterpret_cast<uint8_t*>(p->o);
  a.o_sr = p->o_stride_row;
  a.o_sh = p->o_stride_head;
  a.o_dtype = p->o_dtype;
  a.lse = reinterpret_cast<uint8_t*>(p->lse);
  a.lse_sr = p->lse_stride_row;
  a.lse_dtype = p->lse_dtype;
  a.part_lse = reinterpret_cast<float*>(ws + pl.ws_lse);
  a.part_o = reinterpret_cast<float*>(ws + pl.ws_o);
  a.nsplit = pl.nsplit;
  if (pl.mma) return fp8 ? launch_tree_mma<true>(p, a, pl, ws, st) : launch_tree_mma<false>(p, a, pl, ws, st);
  rc = fp8 ? launch_generic<true>(a, st) : launch_generic<false>(a, st);
  if (rc != QMLA_OK) return rc;
  if (a.nsplit > 1) tree_join_kernel<<<a.reqs * a.nodes * a.heads, 128, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

}  // extern "C"
