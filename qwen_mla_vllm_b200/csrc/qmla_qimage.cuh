// Query rows as the tensor cores read them: K-major operand images with the 128-byte swizzle,
// written to the workspace once per call so that a kernel stages a whole image with bulk copies.
//
// An image holds `nrows` rows (a multiple of 8) of `chunks` 128-byte columns, term by term:
//   byte (term, chunk, row, b) = term * term_bytes + chunk * nrows * 128 + row * 128 + (b ^ ((row & 7) << 4))
// A query element is a sum of up to three terms of the cache's element type, each the rounding of what
// the ones before it leave:
//   bf16 cache: a bf16 query is one term, an f16 query two (8 + 8 bits hold its 11);
//   FP8 cache:  an e4m3 term (4 significant bits) and e5m2 terms (3 bits, down to 2^-16), after a
//               scaling by the power of two that brings the row's largest element into (224, 448].
//               Rounding to nearest leaves a remainder that one e5m2 term holds exactly for a bf16
//               query and two for an f16 query, as long as the e4m3 term is normal: down to 2^-15 of the
//               row's largest element.  Below that an element is off by at most 2^-13 of the scale,
//               2^-21 of the largest element.
// The scaling is undone where the scores are (the caller keeps its inverse).
#pragma once
#include "qmla_decode.cuh"

namespace qmla {

inline int q_terms(bool fp8, int q_dtype) { return (fp8 ? 2 : 1) + (q_dtype == 1 ? 1 : 0); }

// Formats of the terms in a kind::f8f6f4 instruction descriptor.
__device__ __forceinline__ uint32_t q_term_format(int term) { return term == 0 ? 0u : 1u; }

__device__ __forceinline__ uint8_t f32_to_e5m2(float x) {
  return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E5M2);
}
__device__ __forceinline__ float e5m2_to_f32(uint8_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E5M2)));
}

struct QSource {
  const uint8_t *q, *q_pe;
  int64_t q_sr, q_sh, qpe_sr, qpe_sh;  // elements
  int dtype;
  int rank, qk_dim;
  int vec;  // rows may be read in 16-byte units (q_vec)
};

// Rows of q and q_pe start on 16-byte boundaries and hold whole 16-byte units.
inline int q_vec(const void* q, int64_t sr, int64_t sh, const void* pe, int64_t psr, int64_t psh, int rank, int qk_dim) {
  auto ok = [](const void* p, int64_t a, int64_t b) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a % 8 == 0 && b % 8 == 0;
  };
  return ok(q, sr, sh) && ok(pe, psr, psh) && rank % 8 == 0 && qk_dim % 8 == 0;
}

// Writes one row (all terms) of an image; src_row < 0 writes zeros.  One warp; a lane holds all its
// units (of at most 2048 elements) before it converts any, so their loads overlap.  Returns the
// inverse of the row's scaling in every lane.
template <bool FP8>
__device__ __forceinline__ float write_q_row(const QSource& s, int64_t src_row, int head, uint8_t* img, int row,
                                             int nrows, int chunks, int terms) {
  constexpr int V = FP8 ? 16 : 8;        // elements of a 16-byte unit of the image
  constexpr int U = 2048 / V / 32;       // units per lane at most
  const int lane = threadIdx.x & 31;
  const int units = chunks * 8;
  const int64_t term_bytes = (int64_t)chunks * nrows * 128;
  const uint8_t* q = s.q + (src_row * s.q_sr + (int64_t)head * s.q_sh) * 2;
  const uint8_t* pe = s.q_pe + (src_row * s.qpe_sr + (int64_t)head * s.qpe_sh - s.rank) * 2;
  uint4 raw[U][V / 8];
#pragma unroll
  for (int k = 0; k < U; ++k) {
#pragma unroll
    for (int g = 0; g < V / 8; ++g) {
      const int d = (lane + 32 * k) * V + 8 * g;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (src_row >= 0 && d < s.qk_dim) {
        if (s.vec) {
          v = __ldg(reinterpret_cast<const uint4*>((d < s.rank ? q : pe) + (int64_t)d * 2));
        } else {
          uint16_t e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            e[i] = d + i < s.qk_dim ? __ldg(reinterpret_cast<const uint16_t*>((d + i < s.rank ? q : pe) + (int64_t)(d + i) * 2)) : 0;
          v = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                         e[6] | (uint32_t)e[7] << 16);
        }
      }
      raw[k][g] = v;
    }
  }
  const bool bf = s.dtype == 0;
  auto unpack = [&](const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t lo = (uint16_t)w[i], hi = (uint16_t)(w[i] >> 16);
      f[2 * i] = bf ? __bfloat162float(__ushort_as_bfloat16(lo)) : __half2float(__ushort_as_half(lo));
      f[2 * i + 1] = bf ? __bfloat162float(__ushort_as_bfloat16(hi)) : __half2float(__ushort_as_half(hi));
    }
  };
  float scale = 1.f;
  if constexpr (FP8) {
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int g = 0; g < V / 8; ++g) {
        float f[8];
        unpack(raw[k][g], f);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (fabsf(f[i]) <= 3.0e38f) mx = fmaxf(mx, fabsf(f[i]));  // finite ones
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (mx > 0.f) {
      const int e = max(-100, min(100, (int)floorf(log2f(448.f / mx))));
      scale = exp2f((float)e);
      if (mx * scale > 448.f) scale *= 0.5f;  // log2f may round up to a whole number
    }
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = lane + 32 * k;
    if (u >= units) break;
    float v[V];
#pragma unroll
    for (int g = 0; g < V / 8; ++g) unpack(raw[k][g], v + 8 * g);
    const int64_t at = (int64_t)(u >> 3) * nrows * 128 + row * 128 + (((u & 7) ^ (row & 7)) << 4);
    for (int t = 0; t < terms; ++t) {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (FP8) {
          if (t == 0) v[e] *= scale;
          const bool fin = fabsf(v[e]) <= 448.f;  // not finite: NaN
          const uint8_t b = !fin ? 0x7f : t == 0 ? f32_to_e4m3(v[e]) : f32_to_e5m2(v[e]);
          w[e >> 2] |= (uint32_t)b << (8 * (e & 3));
          v[e] -= t == 0 ? e4m3_to_f32(b) : e5m2_to_f32(b);
        } else {
          const __nv_bfloat16 b = __float2bfloat16_rn(v[e]);
          w[e >> 1] |= (uint32_t)__bfloat16_as_ushort(b) << (16 * (e & 1));
          v[e] = isfinite(v[e]) ? v[e] - __bfloat162float(b) : 0.f;
        }
      }
      *reinterpret_cast<uint4*>(img + t * term_bytes + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  return 1.f / scale;
}

// Byte range of an image as bulk copies of at most 32 KB onto one barrier (its bytes are armed
// by the caller): one lane.
__device__ __forceinline__ void load_image(uint32_t dst, const uint8_t* src, uint32_t bytes, uint32_t bar,
                                           uint64_t policy) {
  for (uint32_t o = 0; o < bytes; o += 32768u) bulk_load_1d(dst + o, src + o, min(32768u, bytes - o), bar, policy);
}

}  // namespace qmla
