// Rotary positions, and the write of a step's rotated keys into the paged latent cache.
//
// Pair i of a token at position p turns by the angle 2 pi * frac(p * step_i): step_i is the
// pair's angular frequency in turns per position, held as a 64-bit binary fraction.  The product
// p * step_i modulo 2^64 is the phase itself, exact to 2^-53 of the frequency at every position
// (p * frequency in 32-bit floats is off by up to 2^-24 * p turns' worth: 0.016 rad at 262,144).
// Its top 32 bits, taken as a signed fraction in [-1/2, 1/2), go to sincospif.
//   (a, b) -> scale * (a cos - b sin, b cos + a sin)        the adjoint turns the other way
// These kernels move bytes (2 or 3 flops per byte): every element is read once and written once, a
// block's sines are computed once for all the heads it rotates, and a block walks up to four token groups
// with the next one's bytes on their way.  Measured on a B200 (copy bandwidth 6.55 TB/s): 32,768 tokens'
// worth of bf16 pairs side by side 106 us, 3.8 TB/s (one group per block: 128 us); 16,384 tokens into an
// FP8 cache, queries in place, 117 us, 3.5 TB/s.  What is left is the turning itself: the update's SMs
// are 75% busy with two-byte shared loads and stores (halves start at odd offsets), DRAM 38%.
// Resident warps count most there: eight blocks of 256 threads (32 registers, a few spilled words in the
// unaligned forms) 117 us, six 156, five 158, two (unbounded registers, four pairs in flight) 209.
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

constexpr int kRotThreads = 256;
constexpr int kRotBlocks = 8;  // of them resident on an SM
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kMaxRot = 512;            // dims of one rotated block
constexpr int kStageBytes = 16 * 1024;  // one staged segment at most
constexpr int kWalk = 4;  // token groups (or tokens) of a block in a long call
constexpr int kBlockBytes = 12 * 1024;  // what a block stages at a time, where a segment is no larger

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

// Quotients of small numbers by a launch constant: exact for n * d < 2^32.
struct FastDiv {
  uint32_t d, magic;
  __host__ static FastDiv of(uint32_t d) { return FastDiv{d, d > 1 ? (uint32_t)(((1ull << 32) + d - 1) / d) : 0u}; }
  __device__ __forceinline__ int div(int n) const { return d > 1 ? (int)__umulhi((uint32_t)n, magic) : n; }
};

// One rotated span of a token: `segs` segments (heads) of `len` elements, each a run of
// heads of `period` dims whose dims [start, start + blocks * rot) turn, rot at a time.
struct RotSpan {
  const uint8_t* x;
  uint8_t* out;
  int64_t x_st, x_ss, o_st, o_ss;  // bytes per token, per segment
  int segs, len, period, start, rot, blocks;
  // units of a segment, segments of a block, pairs and rotated blocks of a head, rotated blocks of a token
  FastDiv by_units, by_segs, by_half, by_blocks, by_items;
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

// (cos, sin) of pair i at a position, scaled; the adjoint turns the other way.
__device__ __forceinline__ float2 turn_of(const RotAngles& g, int64_t pos, int i) {
  const uint64_t phase = (uint64_t)pos * (uint64_t)__ldg(reinterpret_cast<const long long*>(g.steps) + i);
  const float t = (float)(int32_t)(phase >> 32) * 4.656612873077393e-10f;  // 2^-31: half turns
  float s, c;
  sincospif(t, &s, &c);
  return make_float2(c * g.scale, s * (g.adjoint ? -g.scale : g.scale));
}

// Window pair j -> (offset of its first element in a head, pair of its block).
__device__ __forceinline__ uint32_t pair_entry(const RotSpan& s, int interleaved, int j) {
  const int half = s.rot >> 1, blk = s.by_half.div(j), i = j - blk * half;
  return (uint32_t)(s.start + blk * s.rot + (interleaved ? 2 * i : i)) | (uint32_t)i << 16;
}

// Segments [seg0, seg0 + nseg) of tokens [tok0, tok0 + ntok) by way of shared memory: loaded and stored
// in whole 16-byte units (VEC) whatever the window's alignment (58 dims turn as halves of 29), turned in
// place in between.  Every element is staged before any is
// written, so out may be x itself.
template <typename T, bool VEC>
struct Staged {
  static constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  const RotSpan& s;
  uint8_t* stage;
  int64_t tok0;
  int ntok, seg0, nseg;

  __device__ __forceinline__ int total() const { return ntok * nseg * (s.len / V); }
  __device__ __forceinline__ int64_t offset(int u, int64_t st, int64_t ss) const {
    const int r = s.by_units.div(u), k = u - r * (s.len / V);
    const int t = ntok == 1 ? 0 : s.by_segs.div(r), sg = r - t * nseg;
    return (tok0 + t) * st + (int64_t)(seg0 + sg) * ss + (int64_t)k * V * sizeof(T);
  }
  // starts the loads; what the caller does before turn() overlaps them
  __device__ __forceinline__ void load() const {
    const int n = total();
    for (int u = threadIdx.x; u < n; u += kRotThreads) {
      const uint8_t* p = s.x + offset(u, s.x_st, s.x_ss);
      if constexpr (VEC)
        cp_async_16(smem_u32(stage) + 16 * u, p, 16);
      else
        reinterpret_cast<T*>(stage)[u] = *reinterpret_cast<const T*>(p);
    }
  }
  // turns: [ntok][rot / 2], made visible with the staged elements by a barrier
  __device__ __forceinline__ void turn(int interleaved, const float2* turns) const {
    const bool even = ((s.start | s.period) & 1) == 0;
    if (interleaved && even)
      turn_as<2>(1, turns);
    else if (!interleaved && even && (s.rot & 3) == 0)
      turn_as<1>(s.rot >> 1, turns);
    else
      turn_as<0>(interleaved ? 1 : s.rot >> 1, turns);
    store();
  }
  // A lane keeps its pairs (their sines in registers while the block holds one token) and walks the rotated
  // blocks; where a block has fewer pairs than a warp has lanes, the warp takes several at a time.
  // Form 0: a pair as two elements `dist` apart; 1: two neighbouring pairs, a word of each half; 2: a pair
  // that is one word.
  template <int FORM>
  __device__ __forceinline__ void turn_as(int dist, const float2* turns) const {
    constexpr int P = FORM == 1 ? 2 : 1;
    struct alignas(2 * sizeof(T)) Word { T a, b; };
    const int half = s.rot >> 1, lanes = half / P, lane = threadIdx.x & 31;
    const int items = nseg * (s.len / s.period) * s.blocks, all = ntok * items;
    const int share = lanes < 32 ? 32 / lanes : 1, sub = lanes < 32 ? lane / lanes : 0;
    if (sub >= share) return;
    for (int i = P * (lane - sub * lanes); i < half; i += 32 * P) {
      float2 cs[P];
#pragma unroll
      for (int q = 0; q < P; ++q) cs[q] = turns[i + q];
      T* base = reinterpret_cast<T*>(stage) + s.start + (dist == 1 ? 2 * i : i);
      for (int m = (threadIdx.x >> 5) * share + sub; m < all; m += kRotWarps * share) {
        const int row = s.by_blocks.div(m);
        T* at = base + row * s.period + (m - row * s.blocks) * s.rot;
        if (ntok > 1)
#pragma unroll
          for (int q = 0; q < P; ++q) cs[q] = turns[s.by_items.div(m) * half + i + q];
        auto turned = [](float2 c, T& x, T& y) {
          const float fx = to_f32(x), fy = to_f32(y);
          x = from_f32<T>(fx * c.x - fy * c.y);
          y = from_f32<T>(fy * c.x + fx * c.y);
        };
        if constexpr (FORM == 0) {
          turned(cs[0], at[0], at[dist]);
        } else if constexpr (FORM == 1) {
          Word v = *reinterpret_cast<const Word*>(at), w = *reinterpret_cast<const Word*>(at + dist);
          turned(cs[0], v.a, w.a);
          turned(cs[P - 1], v.b, w.b);
          *reinterpret_cast<Word*>(at) = v;
          *reinterpret_cast<Word*>(at + dist) = w;
        } else {
          Word v = *reinterpret_cast<const Word*>(at);
          turned(cs[0], v.a, v.b);
          *reinterpret_cast<Word*>(at) = v;
        }
      }
    }
  }
  __device__ __forceinline__ void store() const {
    __syncthreads();
    const int n = total();
#pragma unroll 2
    for (int u = threadIdx.x; u < n; u += kRotThreads) {
      uint8_t* p = s.out + offset(u, s.o_st, s.o_ss);
      if constexpr (VEC)
        *reinterpret_cast<uint4*>(p) = reinterpret_cast<const uint4*>(stage)[u];
      else
        *reinterpret_cast<T*>(p) = reinterpret_cast<const T*>(stage)[u];
    }
  }
};

// Commits the copies started so far as one group / waits until at most `left` groups are in flight.
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int left>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(left) : "memory");
}

// A block walks the token groups from its own on, gridDim.x apart, the next group's elements on their
// way to the other half of the stage while it turns this one's.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRotThreads, kRotBlocks) rotary_kernel(const RotSpan s, const RotAngles g,
                                                             int64_t n, int tpb, int spb) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int half = s.rot >> 1;
  float2* turns = reinterpret_cast<float2*>(smem);
  uint8_t* stage0 = smem + ((tpb * half * 8 + 15) & ~15);
  const int stage_bytes = (tpb * spb * s.len * (int)sizeof(T) + 15) & ~15;
  const int seg0 = blockIdx.y * spb, nseg = min(spb, s.segs - seg0);
  const int64_t groups = (n + tpb - 1) / tpb;
  auto group = [&](int64_t i, int buf) {
    return Staged<T, VEC>{s, stage0 + buf * stage_bytes, i * tpb, (int)min((int64_t)tpb, n - i * tpb), seg0, nseg};
  };
  group(blockIdx.x, 0).load();
  copies_commit();
  int buf = 0;
  for (int64_t i = blockIdx.x; i < groups; i += gridDim.x, buf ^= 1) {
    const Staged<T, VEC> st = group(i, buf);
    if (i + gridDim.x < groups) group(i + gridDim.x, buf ^ 1).load();
    copies_commit();
    for (int x = threadIdx.x; x < st.ntok * half; x += kRotThreads) {
      const int t = s.by_half.div(x), k = x - t * half;
      turns[x] = turn_of(g, position(g, st.tok0 + t), k);
    }
    copies_wait<1>();
    __syncthreads();
    st.turn(g.interleaved, turns);
    __syncthreads();  // the stage and the sines are free
  }
}

// Pairs side by side within 16-byte units: a thread turns the units it loads, two at a time, the next two
// (of the next token group at the end) on their way before these are turned.  Two units and six resident
// blocks 106 us at the size above; four units and four blocks 111, two and eight (spilling) 123.
template <typename T>
__global__ void __launch_bounds__(kRotThreads, 6) rotary_pairs_kernel(const RotSpan s, const RotAngles g,
                                                                   int64_t n, int tpb, int spb) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int V = 16 / (int)sizeof(T), U = 2;
  float2* turns = reinterpret_cast<float2*>(smem);
  const int half = s.rot >> 1, win = s.blocks * s.rot, ups = s.len / V;
  const int seg0 = blockIdx.y * spb, nseg = min(spb, s.segs - seg0);
  const int64_t groups = (n + tpb - 1) / tpb;
  auto total_of = [&](int64_t i) { return (int)min((int64_t)tpb, n - i * tpb) * nseg * ups; };
  // unit u of group i: its token in the group and its window dim, and its place
  auto place = [&](int64_t i, int u, int& t, int& k) -> int64_t {
    const int r = s.by_units.div(u);
    k = u - r * ups;
    t = tpb == 1 ? 0 : s.by_segs.div(r);
    return seg0 + r - t * nseg;
  };
  uint4 raw[U];
  auto load = [&](int64_t i, int u0) {
    const int total = i < groups ? total_of(i) : 0;
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int u = u0 + q * kRotThreads;
      if (u < total) {
        int t, k;
        const int64_t sg = place(i, u, t, k);
        raw[q] = __ldcs(reinterpret_cast<const uint4*>(s.x + (i * tpb + t) * s.x_st + sg * s.x_ss + (int64_t)k * 16));
      }
    }
  };
  load(blockIdx.x, threadIdx.x);
  for (int64_t i = blockIdx.x; i < groups; i += gridDim.x) {
    const int total = total_of(i), ntok = (int)min((int64_t)tpb, n - i * tpb);
    __syncthreads();  // the sines are free
    for (int x = threadIdx.x; x < ntok * half; x += kRotThreads) {
      const int t = s.by_half.div(x), k = x - t * half;
      turns[x] = turn_of(g, position(g, i * tpb + t), k);
    }
    __syncthreads();
    for (int u0 = threadIdx.x; u0 - (int)threadIdx.x < total; u0 += U * kRotThreads) {
      uint4 cur[U];
#pragma unroll
      for (int q = 0; q < U; ++q) cur[q] = raw[q];
      if (u0 - (int)threadIdx.x + U * kRotThreads < total)
        load(i, u0 + U * kRotThreads);
      else
        load(i + gridDim.x, threadIdx.x);
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int u = u0 + q * kRotThreads;
        if (u < total) {
          int t, k;
          const int64_t sg = place(i, u, t, k);
          T* v = reinterpret_cast<T*>(&cur[q]);
          const float2* tb = turns + t * half;
          const int d0 = k * V - s.start;  // window dim of the unit's first element (even)
          int w = d0 >= 0 && d0 < win ? d0 - 2 * half * s.by_half.div(d0 >> 1) : 0;
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            if (d0 + e >= 0 && d0 + e < win) {
              const float2 cs = tb[w >> 1];
              const float x = to_f32(v[e]), y = to_f32(v[e + 1]);
              v[e] = from_f32<T>(x * cs.x - y * cs.y);
              v[e + 1] = from_f32<T>(y * cs.x + x * cs.y);
              w = w + 2 == s.rot ? 0 : w + 2;
            }
          }
          *reinterpret_cast<uint4*>(s.out + (i * tpb + t) * s.o_st + sg * s.o_ss + (int64_t)k * 16) = cur[q];
        }
      }
    }
  }
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
  int row_blocks, q_blocks;  // blocks that write rows; blocks per part of q
  int64_t n;
};

__device__ __forceinline__ uint8_t e4m3_of(float x) {
  return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// A token's cache row, by one warp: latent, rotated keys, divisors.  An FP8 row rounds x / k_scale once,
// saturating at +-448 (NaN stays NaN), its rotated keys not to bf16 first.
template <bool FP8>
__device__ __forceinline__ void write_row(const RopeCacheArgs& a, int64_t tok) {
  const int lane = threadIdx.x & 31;
  const int64_t slot = __ldg(reinterpret_cast<const long long*>(a.slots) + tok);
  const int half = a.q.rot >> 1, pairs = a.q.blocks * half, dist = a.g.interleaved ? 1 : half;
  const uint8_t* lat = a.latent + tok * a.lat_st;
  const __nv_bfloat16* kp = reinterpret_cast<const __nv_bfloat16*>(a.k_pe + tok * a.kpe_st);
  if (slot < 0) return;  // a padding token: nothing is cached
  if (slot >= a.num_slots) {
    if (lane == 0 && a.status) atomicOr(a.status, QMLA_DEV_ERR_INDEX);
    return;
  }
  const int64_t pos = position(a.g, tok);
  const float inv = FP8 ? 1.0f / __ldg(a.k_scale) : 1.0f;
  uint8_t* dst = a.cache + slot / a.page_size * a.page_b + slot % a.page_size * a.tok_b;
  constexpr int kLoads = FP8 ? 2 : 1;  // 16-byte loads per 16-byte store
  const int units = a.vec_row ? a.rank / (FP8 ? 16 : 8) : 0;
#pragma unroll 2
  for (int u = lane; u < units; u += 32) {
    uint4 lv[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) lv[i] = __ldg(reinterpret_cast<const uint4*>(lat) + kLoads * u + i);
    if constexpr (FP8) {
      const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(lv);
      alignas(16) __nv_fp8x2_storage_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = __bfloat1622float2(b[i]);
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * inv, f.y * inv), __NV_SATFINITE, __NV_E4M3);
      }
      reinterpret_cast<uint4*>(dst)[u] = *reinterpret_cast<const uint4*>(w);
    } else {
      reinterpret_cast<uint4*>(dst)[u] = lv[0];
    }
  }
  if (!a.vec_row) {
    for (int d = lane; d < a.rank; d += 32) {
      const __nv_bfloat16 v = reinterpret_cast<const __nv_bfloat16*>(lat)[d];
      if constexpr (FP8)
        dst[d] = e4m3_of(__bfloat162float(v) * inv);
      else
        reinterpret_cast<__nv_bfloat16*>(dst)[d] = v;
    }
  }
#pragma unroll 2
  for (int j = lane; j < pairs; j += 32) {
    const uint32_t e = pair_entry(a.q, a.g.interleaved, j);
    const int d = e & 0xffffu;
    const float x = __bfloat162float(kp[d]), y = __bfloat162float(kp[d + dist]);
    const float2 cs = turn_of(a.g, pos, e >> 16);
    const float ra = x * cs.x - y * cs.y, rb = y * cs.x + x * cs.y;
    if constexpr (FP8) {
      dst[a.rank + d] = e4m3_of(ra * inv);
      dst[a.rank + d + dist] = e4m3_of(rb * inv);
    } else {
      reinterpret_cast<__nv_bfloat16*>(dst)[a.rank + d] = __float2bfloat16_rn(ra);
      reinterpret_cast<__nv_bfloat16*>(dst)[a.rank + d + dist] = __float2bfloat16_rn(rb);
    }
  }
  // score divisors: as they are (bf16), log2 codes, or raw bf16 bytes
  for (int h = lane; h < a.heads; h += 32) {
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
}

// The first row_blocks blocks write the cache rows, a warp per token; the others rotate q, each one part
// (hpb heads) of tokens q_blocks apart, the next token's heads on their way to the other half of the stage
// while this one's are turned.  No two blocks touch the same bytes, so q may be rotated in place.
template <bool FP8, bool VEC>
__global__ void __launch_bounds__(kRotThreads, kRotBlocks) rope_cache_kernel(const RopeCacheArgs a) {
  if ((int)blockIdx.x < a.row_blocks) {
    const int64_t tok = (int64_t)blockIdx.x * kRotWarps + (threadIdx.x >> 5);
    if (tok < a.n) write_row<FP8>(a, tok);
    return;
  }
  extern __shared__ __align__(16) uint8_t smem[];
  const int half = a.q.rot >> 1;
  float2* turns = reinterpret_cast<float2*>(smem);
  uint8_t* stage0 = smem + ((half * 8 + 15) & ~15);
  const int stage_bytes = (a.hpb * a.q.len * 2 + 15) & ~15;
  const int x = blockIdx.x - a.row_blocks, part = x / a.q_blocks;
  const int seg0 = part * a.hpb;
  auto token = [&](int64_t tok, int buf) {
    return Staged<__nv_bfloat16, VEC>{a.q, stage0 + buf * stage_bytes, tok, 1, seg0, min(a.hpb, a.q.segs - seg0)};
  };
  int64_t tok = x - part * a.q_blocks;
  token(tok, 0).load();
  copies_commit();
  for (int buf = 0; tok < a.n; tok += a.q_blocks, buf ^= 1) {
    const Staged<__nv_bfloat16, VEC> st = token(tok, buf);
    if (tok + a.q_blocks < a.n) token(tok + a.q_blocks, buf ^ 1).load();
    copies_commit();
    for (int i = threadIdx.x; i < half; i += kRotThreads) turns[i] = turn_of(a.g, position(a.g, tok), i);
    copies_wait<1>();
    __syncthreads();
    st.turn(a.g.interleaved, turns);
    __syncthreads();  // the stage and the sines are free
  }
}

template <typename K>
bool room_for(K kernel, size_t smem) {
  return smem <= 48 * 1024 ||
         cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess;
}

// Blocks of a walk over `groups` of work, `parts` blocks side by side on each: up to kWalk groups per
// block, fewer where that would leave less than 16 blocks per SM.
int64_t walk_blocks(int64_t groups, int64_t parts, int sms) {
  const int64_t walk = std::max<int64_t>(1, std::min<int64_t>(kWalk, groups * parts / (16 * (int64_t)sms)));
  return (groups + walk - 1) / walk;
}

bool aligned16(const void* p, int64_t s1, int64_t s2) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s1 % 16 == 0 && s2 % 16 == 0;
}

template <typename T>
int launch_rotary(RotSpan s, const RotAngles& g, int64_t n, bool vec, int tpb, int spb, int sms,
                  cudaStream_t st) {
  const int64_t gx = (n + tpb - 1) / tpb;
  const int gy = (s.segs + spb - 1) / spb;
  if (gx > INT32_MAX || gy > 65535) return QMLA_E_UNSUPPORTED;
  const int half = s.rot / 2;
  s.by_units = FastDiv::of(s.len / (vec ? 16 / (int)sizeof(T) : 1));
  s.by_segs = FastDiv::of(spb);
  s.by_half = FastDiv::of(half);
  s.by_blocks = FastDiv::of(s.blocks);
  s.by_items = FastDiv::of(spb * (s.len / s.period) * s.blocks);
  const size_t head = ((size_t)tpb * half * 8 + 15) / 16 * 16;
  const dim3 grid((unsigned)walk_blocks(gx, gy, sms), gy);
  const size_t stage = 2 * (((size_t)tpb * spb * s.len * sizeof(T) + 15) / 16 * 16);
  auto launch = [&](auto kernel, size_t smem) {
    if (!room_for(kernel, smem)) return (int)QMLA_E_CUDA;
    kernel<<<grid, kRotThreads, smem, st>>>(s, g, n, tpb, spb);
    return cudaGetLastError() == cudaSuccess ? (int)QMLA_OK : (int)QMLA_E_CUDA;
  };
  if (vec && g.interleaved && s.start % 2 == 0 && s.period % (16 / (int)sizeof(T)) == 0)
    return launch(rotary_pairs_kernel<T>, head);
  return vec ? launch(rotary_kernel<T, true>, head + stage) : launch(rotary_kernel<T, false>, head + stage);
}

}  // namespace

extern "C" {

int qmla_rotary(const qmla_rotary_params* p, void* stream) try {
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
  // A block takes about 12 KB (3 units per thread in flight), 4 KB when that leaves SMs idle:
  // several heads of one token, or, where a whole token is less, several tokens.
  const int64_t seg_b = (int64_t)s.len * es;
  int64_t target = kBlockBytes;
  if (p->num_tokens * s.segs * seg_b < 4 * target * di.sms) target = 4096;
  int spb = (int)std::max<int64_t>(1, std::min<int64_t>(s.segs, target / seg_b));
  int tpb = spb == s.segs ? (int)std::max<int64_t>(1, std::min<int64_t>(16, target / (seg_b * s.segs))) : 1;
  tpb = std::max(1, std::min(tpb, 8192 / (s.rot * 4)));  // 8 KB of sines
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == QMLA_DT_BF16) return launch_rotary<__nv_bfloat16>(s, g, p->num_tokens, vec, tpb, spb, di.sms, st);
  if (p->dtype == QMLA_DT_F16) return launch_rotary<__half>(s, g, p->num_tokens, vec, tpb, spb, di.sms, st);
  return launch_rotary<float>(s, g, p->num_tokens, vec, tpb, spb, di.sms, st);
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

int qmla_rope_cache_write(const qmla_rope_cache_params* p, void* stream) try {
  if (!p || p->num_tokens < 0 || p->num_heads < 0 || p->rank <= 0 || p->rope_width <= 0 ||
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
  if ((p->num_heads > 0 && (!p->q_pe || !p->q_out)) || !p->latent || !p->k_pe || !p->positions || !p->slot_mapping || !p->steps ||
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
  // q heads of a block: about 12 KB of them, 4 KB when the tokens alone do not fill the SMs
  const int64_t stage = p->num_tokens >= 2 * di.sms ? kBlockBytes : 4096;
  a.hpb = (int)std::max<int64_t>(1, std::min<int64_t>(p->num_heads, stage / (2 * a.q.len)));
  const int parts = (p->num_heads + a.hpb - 1) / a.hpb;
  if (parts > 65535) return QMLA_E_UNSUPPORTED;
  const int half = a.q.rot / 2;
  a.q.by_units = FastDiv::of(a.q.len / (vec ? 8 : 1));
  a.q.by_segs = FastDiv::of(a.hpb);
  a.q.by_half = FastDiv::of(half);
  a.q.by_blocks = FastDiv::of(a.q.blocks);
  a.q.by_items = FastDiv::of(1);  // a block holds one token
  const size_t smem = ((size_t)half * 8 + 15) / 16 * 16 + 2 * (((size_t)a.hpb * a.q.len * 2 + 15) / 16 * 16);
  a.n = p->num_tokens;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t rows = (a.n + kRotWarps - 1) / kRotWarps, walk = walk_blocks(a.n, parts, di.sms);
  if (rows + walk * parts > INT32_MAX) return QMLA_E_UNSUPPORTED;
  a.row_blocks = (int)rows;
  a.q_blocks = (int)walk;
  auto launch = [&](auto kernel) {
    if (!room_for(kernel, smem)) return (int)QMLA_E_CUDA;
    kernel<<<(unsigned)(rows + walk * parts), kRotThreads, smem, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? (int)QMLA_OK : (int)QMLA_E_CUDA;
  };
  if (fp8) return vec ? launch(rope_cache_kernel<true, true>) : launch(rope_cache_kernel<true, false>);
  return vec ? launch(rope_cache_kernel<false, true>) : launch(rope_cache_kernel<false, false>);
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

}  // extern "C"
