// Rotary positions, and the write of a step's rotated keys into the paged latent cache.
//
// Pair i of a token at position p turns by the angle 2 pi * frac(p * step_i): step_i is the
// pair's angular frequency in turns per position, held as a 64-bit binary fraction.  The product
// p * step_i modulo 2^64 is the phase itself, exact to 2^-53 of the frequency at every position
// (p * frequency in 32-bit floats is off by up to 2^-24 * p turns' worth: 0.016 rad at 262,144).
// Its top 32 bits, taken as a signed fraction in [-1/2, 1/2), go to sincospif.
//   (a, b) -> scale * (a cos - b sin, b cos + a sin)        the adjoint turns the other way
// Both kernels are byte movers bound by HBM (2 or 3 flops per byte): every element is read once
// and written once.  A block's sines are computed once for all the heads it rotates.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstring>

#include "qmla.h"
#include "qmla_host.cuh"
#include "qmla_ptx.cuh"

using namespace qmla;

namespace {

constexpr int kRotThreads = 128;
constexpr int kMaxRot = 512;           // dims of one rotated block
constexpr int kStageBytes = 16 * 1024;  // staged elements of a block at most

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }

// One rotated span of a token: `segs` segments (heads) of `len` elements, each a run of
// heads of `period` dims whose dims [start, start + blocks * rot) turn, rot at a time.
struct RotSpan {
  const uint8_t* x;
  uint8_t* out;
  int64_t x_st, x_ss, o_st, o_ss;  // bytes per token, per segment
  int segs, len, period, start, rot, blocks;
};

struct RotAngles {
  const void* pos;
  int pos_i64;
  const int64_t* steps;
  float scale;
  int interleaved, adjoint;
};

__device__ __forceinline__ int64_t position(const RotAngles& g, int64_t tok) {
  return g.pos_i64 ? __ldg(reinterpret_cast<const long long*>(g.pos) + tok)
                   : (int64_t)__ldg(reinterpret_cast<const int*>(g.pos) + tok);
}

// tab[w] = (cos, signed sin) of window dim w, so that out[w] = x[w] * tab.x + x[partner] * tab.y.
__device__ __forceinline__ void fill_table(float2* tab, const RotAngles& g, int rot, int64_t pos, int i) {
  const uint64_t phase = (uint64_t)pos * (uint64_t)__ldg(reinterpret_cast<const long long*>(g.steps) + i);
  const float t = (float)(int32_t)(phase >> 32) * 4.656612873077393e-10f;  // 2^-31: half turns
  float s, c;
  sincospif(t, &s, &c);
  s *= g.adjoint ? -g.scale : g.scale;
  c *= g.scale;
  const int a = g.interleaved ? 2 * i : i, b = g.interleaved ? 2 * i + 1 : i + rot / 2;
  tab[a] = make_float2(c, -s);
  tab[b] = make_float2(c, s);
}

__device__ __forceinline__ int partner(int w, int rot, int interleaved) {
  const int h = rot >> 1;
  return interleaved ? w ^ 1 : (w < h ? w + h : w - h);
}

// Rotates segments [seg0, seg0 + nseg) of tokens [tok0, tok0 + ntok).  The segments are staged in
// shared memory before any is written: the partner of an element may sit anywhere in the window
// (58 dims turn as halves of 29), so out may be x itself, and global accesses are whole 16-byte
// units (VEC) whatever the window's alignment.  Units belong to a thread in the order they are
// loaded, all loads of a thread in flight at once.
template <typename T, bool VEC>
__device__ __forceinline__ void rotate_segments(const RotSpan& s, int interleaved, const float2* tab,
                                                uint8_t* stage, int64_t tok0, int ntok, int seg0,
                                                int nseg) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  const int ups = s.len / V;  // units per segment
  const int total = ntok * nseg * ups;
  const int win = s.blocks * s.rot;
  const T* st = reinterpret_cast<const T*>(stage);
#pragma unroll 4
  for (int u = threadIdx.x; u < total; u += kRotThreads) {
    const int r = u / ups, k = u - r * ups;
    const int t = r / nseg, sg = r - t * nseg;
    const uint8_t* p = s.x + (tok0 + t) * s.x_st + (int64_t)(seg0 + sg) * s.x_ss + (int64_t)k * V * sizeof(T);
    if constexpr (VEC)
      reinterpret_cast<uint4*>(stage)[u] = *reinterpret_cast<const uint4*>(p);
    else
      reinterpret_cast<T*>(stage)[u] = *reinterpret_cast<const T*>(p);
  }
  __syncthreads();
#pragma unroll 2
  for (int u = threadIdx.x; u < total; u += kRotThreads) {
    const int r = u / ups, k = u - r * ups;
    const int t = r / nseg, sg = r - t * nseg;
    const T* row = st + (int64_t)r * s.len;
    int e = k * V;
    int head = e / s.period;
    int d = e - head * s.period;
    int w = d - s.start;  // dim of the window, then of its block
    if (w >= 0 && w < win) w %= s.rot;
    const float2* tb = tab + t * s.rot;
    alignas(16) T v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const T own = row[e];
      if (d >= s.start && d < s.start + win) {
        const float2 cs = tb[w];
        const float other = to_f32(row[e - w + partner(w, s.rot, interleaved)]);
        v[i] = from_f32<T>(to_f32(own) * cs.x + other * cs.y);
      } else {
        v[i] = own;
      }
      ++e;
      if (++d == s.period) {
        d = 0;
        w = -s.start;
      } else if (++w == s.rot) {
        w = 0;
      }
    }
    uint8_t* p = s.out + (tok0 + t) * s.o_st + (int64_t)(seg0 + sg) * s.o_ss + (int64_t)k * V * sizeof(T);
    if constexpr (VEC)
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
    else
      *reinterpret_cast<T*>(p) = v[0];
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotSpan s, const RotAngles g,
                                                             int64_t n, int tpb, int spb) {
  extern __shared__ __align__(16) uint8_t smem[];
  float2* tab = reinterpret_cast<float2*>(smem);
  uint8_t* stage = smem + ((tpb * s.rot * 8 + 15) & ~15);
  const int64_t tok0 = (int64_t)blockIdx.x * tpb;
  const int ntok = (int)min((int64_t)tpb, n - tok0);
  const int seg0 = blockIdx.y * spb, nseg = min(spb, s.segs - seg0);
  const int half = s.rot >> 1;
  for (int i = threadIdx.x; i < ntok * half; i += kRotThreads) {
    const int t = i / half, k = i - t * half;
    fill_table(tab + t * s.rot, g, s.rot, position(g, tok0 + t), k);
  }
  rotate_segments<T, VEC>(s, g.interleaved, tab, stage, tok0, ntok, seg0, nseg);
}

struct RopeCacheArgs {
  RotSpan q;
  RotAngles g;
  const uint8_t* latent;
  const uint8_t* k_pe;
  int64_t lat_st, kpe_st;  // bytes per token
  const int64_t* slots;
  uint8_t* cache;
  int64_t page_b, tok_b, num_slots;
  int page_size;
  int rank, win, heads, rms_mode;
  int vec_row;  // the latent part moves in 16-byte units
  const float* k_scale;
  int* status;
  int hpb;  // heads per block
};

__device__ __forceinline__ uint8_t e4m3_of(float x) {
  return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// One block per (token, part): part 0 writes the token's cache row, parts 1.. rotate hpb heads of
// q each.  Two parts never touch the same bytes, so q may be rotated in place.
template <bool FP8, bool VEC>
__global__ void __launch_bounds__(kRotThreads) rope_cache_kernel(const RopeCacheArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  float2* tab = reinterpret_cast<float2*>(smem);
  uint8_t* stage = smem + ((a.q.rot * 8 + 15) & ~15);
  const int64_t tok = blockIdx.x;
  const int tid = threadIdx.x;
  for (int i = tid; i < (a.q.rot >> 1); i += kRotThreads)
    fill_table(tab, a.g, a.q.rot, position(a.g, tok), i);
  if (blockIdx.y > 0) {
    const int seg0 = ((int)blockIdx.y - 1) * a.hpb;
    rotate_segments<__nv_bfloat16, VEC>(a.q, a.g.interleaved, tab, stage, tok, 1, seg0,
                                        min(a.hpb, a.q.segs - seg0));
    return;
  }
  const int64_t slot = __ldg(reinterpret_cast<const long long*>(a.slots) + tok);
  if (slot < 0) return;  // padding token: nothing is cached
  if (slot >= a.num_slots) {
    if (tid == 0 && a.status) atomicOr(a.status, QMLA_DEV_ERR_INDEX);
    return;
  }
  uint8_t* dst = a.cache + slot / a.page_size * a.page_b + slot % a.page_size * a.tok_b;
  const uint8_t* lat = a.latent + tok * a.lat_st;
  const __nv_bfloat16* kp = reinterpret_cast<const __nv_bfloat16*>(a.k_pe + tok * a.kpe_st);
  const float inv = FP8 ? 1.0f / __ldg(a.k_scale) : 1.0f;
  // latent: FP8 rows round x / k_scale once, saturating at +-448 (NaN stays NaN)
  if (a.vec_row) {
    if constexpr (FP8) {
      for (int u = tid; u < a.rank / 16; u += kRotThreads) {
        const uint4 v[2] = {reinterpret_cast<const uint4*>(lat)[2 * u], reinterpret_cast<const uint4*>(lat)[2 * u + 1]};
        const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(v);
        alignas(16) __nv_fp8x2_storage_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 f = __bfloat1622float2(b[i]);
          w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * inv, f.y * inv), __NV_SATFINITE, __NV_E4M3);
        }
        reinterpret_cast<uint4*>(dst)[u] = *reinterpret_cast<const uint4*>(w);
      }
    } else {
      for (int u = tid; u < a.rank / 8; u += kRotThreads)
        reinterpret_cast<uint4*>(dst)[u] = reinterpret_cast<const uint4*>(lat)[u];
    }
  } else {
    for (int d = tid; d < a.rank; d += kRotThreads) {
      const __nv_bfloat16 v = reinterpret_cast<const __nv_bfloat16*>(lat)[d];
      if constexpr (FP8)
        dst[d] = e4m3_of(__bfloat162float(v) * inv);
      else
        reinterpret_cast<__nv_bfloat16*>(dst)[d] = v;
    }
  }
  // score divisors: as they are (bf16), log2 codes, or raw bf16 bytes
  for (int h = tid; h < a.heads; h += kRotThreads) {
    const __nv_bfloat16 rb = kp[a.win + h];
    if constexpr (!FP8) {
      reinterpret_cast<__nv_bfloat16*>(dst)[a.rank + a.win + h] = rb;
    } else if (a.rms_mode == QMLA_RMS_LOG8) {
      const float r = fmaxf(__bfloat162float(rb), 1e-30f);
      const float code = (log2f(r) - (-3.0f)) * (255.0f / 6.0f);
      dst[a.rank + a.win + h] = (uint8_t)fminf(fmaxf(rintf(code), 0.f), 255.f);
    } else {
      const uint16_t bits = __bfloat16_as_ushort(rb);
      dst[a.rank + a.win + 2 * h] = (uint8_t)(bits & 0xFF);
      dst[a.rank + a.win + 2 * h + 1] = (uint8_t)(bits >> 8);
    }
  }
  __syncthreads();  // the sines
  // rope keys: an FP8 row rounds the rotated value once (not to bf16 first)
  for (int e = tid; e < a.win; e += kRotThreads) {
    const int w = e % a.q.rot;
    const float2 cs = tab[w];
    const float y = __bfloat162float(kp[e]) * cs.x +
                    __bfloat162float(kp[e - w + partner(w, a.q.rot, a.g.interleaved)]) * cs.y;
    if constexpr (FP8)
      dst[a.rank + e] = e4m3_of(y * inv);
    else
      reinterpret_cast<__nv_bfloat16*>(dst)[a.rank + e] = __float2bfloat16_rn(y);
  }
}

bool aligned16(const void* p, int64_t s1, int64_t s2) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s1 % 16 == 0 && s2 % 16 == 0;
}

template <typename T>
int launch_rotary(const RotSpan& s, const RotAngles& g, int64_t n, bool vec, int tpb, int spb,
                  cudaStream_t st) {
  const int64_t gx = (n + tpb - 1) / tpb;
  const int gy = (s.segs + spb - 1) / spb;
  if (gx > INT32_MAX || gy > 65535) return QMLA_E_UNSUPPORTED;
  const size_t smem = ((size_t)tpb * s.rot * 8 + 15) / 16 * 16 + (size_t)tpb * spb * s.len * sizeof(T);
  if (vec)
    rotary_kernel<T, true><<<dim3((unsigned)gx, gy), kRotThreads, smem, st>>>(s, g, n, tpb, spb);
  else
    rotary_kernel<T, false><<<dim3((unsigned)gx, gy), kRotThreads, smem, st>>>(s, g, n, tpb, spb);
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
}

}  // namespace

extern "C" {

int qmla_rotary(const qmla_rotary_params* p, void* stream) {
  if (!p || p->num_tokens < 0 || p->num_heads <= 0 || p->head_dim <= 0 || p->start < 0 ||
      p->rot_dim < 2 || p->rot_dim % 2 != 0 || p->blocks < 1)
    return QMLA_E_INVALID;
  if (p->dtype != QMLA_DT_BF16 && p->dtype != QMLA_DT_F16 && p->dtype != QMLA_DT_F32)
    return QMLA_E_UNSUPPORTED;
  if (p->rot_dim > kMaxRot) return QMLA_E_UNSUPPORTED;
  if ((int64_t)p->start + (int64_t)p->blocks * p->rot_dim > p->head_dim) return QMLA_E_INVALID;
  if (p->num_tokens == 0) return QMLA_OK;
  if (!p->x || !p->out || !p->positions || !p->steps) return QMLA_E_INVALID;
  const int es = p->dtype == QMLA_DT_F32 ? 4 : 2;
  if ((int64_t)p->head_dim * es > kStageBytes) return QMLA_E_UNSUPPORTED;
  const DevInfo di = dev_info(p->device);
  if (!di.ok) return QMLA_E_CUDA;
  DeviceGuard dg(p->device);
  if (!dg.ok()) return QMLA_E_CUDA;
  RotSpan s;
  s.x = reinterpret_cast<const uint8_t*>(p->x);
  s.out = reinterpret_cast<uint8_t*>(p->out);
  s.x_st = p->x_stride_token * es;
  s.x_ss = p->x_stride_head * es;
  s.o_st = p->out_stride_token * es;
  s.o_ss = p->out_stride_head * es;
  s.segs = p->num_heads;
  s.len = s.period = p->head_dim;
  s.start = p->start;
  s.rot = p->rot_dim;
  s.blocks = p->blocks;
  if (s.x == s.out && s.x_st == s.o_st && s.x_ss == s.o_ss) {
    // in place: only the window is read and written
    s.x += (int64_t)s.start * es;
    s.out += (int64_t)s.start * es;
    s.len = s.period = s.blocks * s.rot;
    s.start = 0;
  }
  auto ok16 = [&](const RotSpan& r) {
    return (int64_t)r.len * es % 16 == 0 && aligned16(r.x, r.x_st, r.x_ss) && aligned16(r.out, r.o_st, r.o_ss);
  };
  bool vec = ok16(s);
  if (!vec && s.x_ss == (int64_t)s.len * es && s.o_ss == s.x_ss && s.x_ss * s.segs <= kStageBytes) {
    // heads packed side by side whose width is not a multiple of 16 bytes: a whole token's is
    RotSpan f = s;
    f.len = s.len * s.segs;
    f.segs = 1;
    f.x_ss = f.o_ss = 0;
    if (ok16(f)) {
      s = f;
      vec = true;
    }
  }
  const RotAngles g{p->positions, p->positions_i64 != 0, p->steps, p->scale, p->interleaved != 0, p->adjoint != 0};
  // A block takes about 8 KB (4 units per thread in flight), 2 KB when that leaves SMs idle:
  // several heads of one token, or, where a whole token is less, several tokens.
  const int64_t seg_b = (int64_t)s.len * es;
  int64_t target = 8192;
  if (p->num_tokens * s.segs * seg_b < 2 * target * di.sms) target = 2048;
  int spb = (int)std::max<int64_t>(1, std::min<int64_t>(s.segs, target / seg_b));
  int tpb = spb == s.segs ? (int)std::max<int64_t>(1, std::min<int64_t>(16, target / (seg_b * s.segs))) : 1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == QMLA_DT_BF16) return launch_rotary<__nv_bfloat16>(s, g, p->num_tokens, vec, tpb, spb, st);
  if (p->dtype == QMLA_DT_F16) return launch_rotary<__half>(s, g, p->num_tokens, vec, tpb, spb, st);
  return launch_rotary<float>(s, g, p->num_tokens, vec, tpb, spb, st);
}

int qmla_rope_cache_write(const qmla_rope_cache_params* p, void* stream) {
  if (!p || p->num_tokens < 0 || p->num_heads <= 0 || p->rank <= 0 || p->rope_width <= 0 ||
      p->rms_heads < 0 || p->rot_dim < 2 || p->rot_dim % 2 != 0 || p->rope_width % p->rot_dim != 0 ||
      p->page_size <= 0 || p->num_pages < 0)
    return QMLA_E_INVALID;
  if (p->rot_dim > kMaxRot || (int64_t)p->rope_width * 2 > kStageBytes) return QMLA_E_UNSUPPORTED;
  const bool fp8 = p->kv_dtype == QMLA_DT_FP8E4M3;
  if (!fp8 && p->kv_dtype != QMLA_DT_BF16) return QMLA_E_UNSUPPORTED;
  if (fp8 ? (p->rms_mode != QMLA_RMS_LOG8 && p->rms_mode != QMLA_RMS_BF16 && p->rms_mode != QMLA_RMS_NONE)
          : (p->rms_mode != QMLA_RMS_NATIVE && p->rms_mode != QMLA_RMS_NONE))
    return QMLA_E_INVALID;
  const int heads = p->rms_mode == QMLA_RMS_NONE ? 0 : p->rms_heads;
  const int es = fp8 ? 1 : 2;
  const int tail = heads * (p->rms_mode == QMLA_RMS_BF16 ? 2 : 1);
  if (p->kv_row_width < (int64_t)p->rank + p->rope_width + tail || p->kv_stride_token < p->kv_row_width)
    return QMLA_E_INVALID;
  if (p->num_tokens == 0) return QMLA_OK;
  if (p->num_tokens > INT32_MAX) return QMLA_E_UNSUPPORTED;
  if (!p->q_pe || !p->q_out || !p->latent || !p->k_pe || !p->positions || !p->slot_mapping || !p->steps ||
      !p->kv_cache || (fp8 && !p->k_scale))
    return QMLA_E_INVALID;
  const DevInfo di = dev_info(p->device);
  if (!di.ok) return QMLA_E_CUDA;
  DeviceGuard dg(p->device);
  if (!dg.ok()) return QMLA_E_CUDA;
  RopeCacheArgs a;
  memset(&a, 0, sizeof(a));
  a.q.x = reinterpret_cast<const uint8_t*>(p->q_pe);
  a.q.out = reinterpret_cast<uint8_t*>(p->q_out);
  a.q.x_st = p->q_stride_token * 2;
  a.q.x_ss = p->q_stride_head * 2;
  a.q.o_st = p->q_out_stride_token * 2;
  a.q.o_ss = p->q_out_stride_head * 2;
  a.q.segs = p->num_heads;
  a.q.len = a.q.period = p->rope_width;
  a.q.start = 0;
  a.q.rot = p->rot_dim;
  a.q.blocks = p->rope_width / p->rot_dim;
  a.g = RotAngles{p->positions, p->positions_i64 != 0, p->steps, p->scale, p->interleaved != 0, 0};
  a.latent = reinterpret_cast<const uint8_t*>(p->latent);
  a.k_pe = reinterpret_cast<const uint8_t*>(p->k_pe);
  a.lat_st = p->latent_stride * 2;
  a.kpe_st = p->k_pe_stride * 2;
  a.slots = p->slot_mapping;
  a.cache = reinterpret_cast<uint8_t*>(p->kv_cache);
  a.page_b = p->kv_stride_page * es;
  a.tok_b = p->kv_stride_token * es;
  a.num_slots = (int64_t)p->num_pages * p->page_size;
  a.page_size = p->page_size;
  a.rank = p->rank;
  a.win = p->rope_width;
  a.heads = heads;
  a.rms_mode = p->rms_mode;
  a.k_scale = p->k_scale;
  a.status = p->status;
  a.vec_row = aligned16(a.latent, a.lat_st, 0) && aligned16(a.cache, a.page_b, a.tok_b) && p->rank % (fp8 ? 16 : 8) == 0;
  const bool vec = a.q.len * 2 % 16 == 0 && aligned16(a.q.x, a.q.x_st, a.q.x_ss) && aligned16(a.q.out, a.q.o_st, a.q.o_ss);
  // q heads of a block: about 4 KB of them
  a.hpb = std::max(1, std::min(p->num_heads, 4096 / (2 * a.q.len)));
  const int parts = 1 + (p->num_heads + a.hpb - 1) / a.hpb;
  if (parts > 65535) return QMLA_E_UNSUPPORTED;
  const size_t smem = ((size_t)a.q.rot * 8 + 15) / 16 * 16 + (size_t)a.hpb * a.q.len * 2;
  const dim3 grid((unsigned)p->num_tokens, parts);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (fp8)
    vec ? rope_cache_kernel<true, true><<<grid, kRotThreads, smem, st>>>(a)
        : rope_cache_kernel<true, false><<<grid, kRotThreads, smem, st>>>(a);
  else
    vec ? rope_cache_kernel<false, true><<<grid, kRotThreads, smem, st>>>(a)
        : rope_cache_kernel<false, false><<<grid, kRotThreads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
}

}  // extern "C"
