// Accumulated attention weight of every cached token.
//
//   weights[r][t] = decay * weights[r][t] + sum over request r's query rows (j, h) of exp(s_jht - lse_jh)
//   s_jht = (q_jh . k_t) / rms_th * sm_scale
//
// for the tokens t before the longest of the request's row lengths.  lse is what the decode of the
// same queries returned, so nothing is normalised here: one pass over the keys, one number per
// token out.  Rows whose lse is not finite (nothing visible) add nothing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstring>

#include "qmla.h"
#include "qmla_decode.cuh"
#include "qmla_host.cuh"

using namespace qmla;

namespace {

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

}  // namespace

extern "C" {

int qmla_weights_workspace_bytes(const qmla_weights_params* p, int64_t* bytes) {
  if (!bytes) return QMLA_E_INVALID;
  const int rc = check_params(p);
  if (rc != QMLA_OK) return rc;
  *bytes = 0;
  return QMLA_OK;
}

int qmla_accumulate_weights(const qmla_weights_params* p, void* stream) {
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
  const dim3 grid((unsigned)std::max(1, 8 * di.sms / p->num_reqs), p->num_reqs);
  if (fp8)
    weights_generic_kernel<true><<<grid, 256, 0, st>>>(a);
  else
    weights_generic_kernel<false><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
}

}  // extern "C"
