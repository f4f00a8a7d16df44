// Eviction from the paged latent cache by accumulated attention weight.
//
// Of request r's n tokens the K = min(n, budget) with the largest weights stay (protected ones before
// all others, ties to the lowest index).  The cache is closed up by moving as few rows as possible: the
// kept tokens at K and beyond move, in ascending order, into the places below K that were given up, in
// ascending order.  Sources lie at or above K and destinations below it, so no order among the
// moves matters, and a kept token below K never moves.  Order in the cache means nothing to the
// attention (keys carry their rotation); `positions` remembers each token's own.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

#include "qmla.h"
#include "qmla_host.cuh"

namespace cg = cooperative_groups;
using namespace qmla;

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;          // 11, 11 and 10 bits of the key per pass
constexpr int kMaxKeys = 40 * 1024;  // keys of a CTA kept in shared memory
constexpr int kMaxCluster = 8;       // CTAs of one request

struct EvictArgs {
  const float* w;
  int64_t w_sr;
  const int32_t* pos;
  int64_t pos_sr;
  int64_t cols;  // columns of weights and positions
  const int32_t* lens;
  const int32_t* budgets;  // per request, or null
  int budget;
  int sinks;
  const int32_t* recent_from;  // per request, or null
  float* new_w;
  int32_t* new_p;
  int64_t new_sr, new_cols;
  int32_t* new_lens;
  int32_t *src, *dst, *count;  // workspace: [reqs][move_cols] lists, [reqs]
  int64_t move_cols;
  int reqs;
  uint8_t* cache;
  int64_t page_b, tok_b, num_pages, row_b;
  const int32_t* bt;
  int64_t bt_stride, bt_cols;
  int page_size;
  int vec;  // rows move in 16-byte units
  int keys_fit;
};

__device__ __forceinline__ int64_t tokens_of(const EvictArgs& a, int r) {
  const int64_t n = max(__ldg(a.lens + r), 0);
  return min(n, min(a.cols, a.bt_cols * a.page_size));
}
__device__ __forceinline__ int64_t kept_of(const EvictArgs& a, int r, int64_t n) {
  int b = a.budget;
  if (a.budgets) b = min(b, __ldg(a.budgets + r));
  return min(n, (int64_t)max(b, 0));
}

// Order-preserving 32-bit key of a token: protected tokens above everything, NaN weights below.
__device__ __forceinline__ uint32_t key_of(const EvictArgs& a, int r, int64_t t, int recent) {
  const int p = __ldg(a.pos + r * a.pos_sr + t);
  if (p < a.sinks || (a.recent_from && p >= recent)) return 0xffffffffu;
  const float f = __ldg(a.w + r * a.w_sr + t) + 0.0f;  // -0 counts as 0
  if (f != f) return 0u;
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sum over the cluster's warps of a value given by all lanes of each (two 32-bit sums side by
// side in 64 bits).  cta_box: this scan's own place in shared memory, so that no barrier has to
// follow before it is used again; the caller's next cluster barrier keeps it alive.
__device__ __forceinline__ uint64_t cluster_scan(cg::cluster_group& cl, uint64_t* warp_box, uint64_t* cta_box, uint64_t v) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // warp_box is free
  if (lane == 0) warp_box[warp] = v;
  __syncthreads();
  if (warp == 0) {
    uint64_t x = warp_box[lane];
    const uint64_t own = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    warp_box[lane] = x - own;
    if (lane == 31) *cta_box = x;
  }
  cl.sync();
  uint64_t base = warp_box[warp];
#pragma unroll
  for (int c = 0; c < kMaxCluster; ++c)
    if (c < (int)cl.block_rank()) base += *cl.map_shared_rank(cta_box, c);
  return base;
}

// One cluster per request.  The K-th largest key by three radix passes over histograms that the
// cluster's CTAs add up through distributed shared memory; then the tokens equal to it, the
// movers and the holes are numbered in index order (each warp owns a contiguous run of tokens).
// A request's keys are read from memory once and stay in shared memory.
// Bound by its chain of passes over the keys (three histograms, two numbered walks), not by bytes: 50 us for 16
// requests of up to 65,536 tokens (eight CTAs each, a cluster barrier per pass), 15 us for 4 of up to 2048, where a
// request is one CTA with two keys per thread and no peer to wait for.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ int hists[3][kBins];  // one per pass: none is cleared while the peers may still read it
  __shared__ int warp_sum[kSelWarps];
  __shared__ uint64_t warp_box[kSelWarps], cta_box[2];
  __shared__ int found_bin, found_above;
  cg::cluster_group cl = cg::this_cluster();
  const int C = cl.num_blocks(), rank = cl.block_rank();
  const int r = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t n = tokens_of(a, r), K = kept_of(a, r, n);
  const int recent = a.recent_from ? __ldg(a.recent_from + r) : 0;
  // the output columns past the kept ones
  for (int64_t t = K + rank * kSelThreads + tid; t < a.new_cols; t += (int64_t)C * kSelThreads) {
    a.new_w[r * a.new_sr + t] = 0.f;
    a.new_p[r * a.new_sr + t] = -1;
  }
  if (rank == 0 && tid == 0) a.new_lens[r] = (int)K;
  if (K == n || K == 0) {  // the same for the whole cluster: nothing moves
    for (int64_t t = rank * kSelThreads + tid; t < K; t += (int64_t)C * kSelThreads) {
      a.new_w[r * a.new_sr + t] = __ldg(a.w + r * a.w_sr + t);
      a.new_p[r * a.new_sr + t] = __ldg(a.pos + r * a.pos_sr + t);
    }
    if (rank == 0 && tid == 0) a.count[r] = 0;
    return;
  }
  const int64_t lo = n * rank / C, hi = n * (rank + 1) / C;
  const int m = (int)(hi - lo);
  auto key_at = [&](int i) { return a.keys_fit ? keys[i] : key_of(a, r, lo + i, recent); };
  if (a.keys_fit) {
#pragma unroll 4
    for (int i = tid; i < m; i += kSelThreads) keys[i] = key_of(a, r, lo + i, recent);
  }
  for (int b = tid; b < 3 * kBins; b += kSelThreads) (&hists[0][0])[b] = 0;
  __syncthreads();
  uint32_t prefix = 0;  // the bits of the K-th largest key found so far
  int64_t want = K;     // its rank among the keys that share them
  int shift = 32;
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass == 2 ? 10 : 11;
    const uint32_t above = pass == 0 ? 0u : 0xffffffffu << shift;  // bits that are fixed
    shift -= bits;
    const uint32_t mask = (1u << bits) - 1;
    int* hist = hists[pass];
#pragma unroll 4
    for (int i = tid; i < m; i += kSelThreads) {
      const uint32_t k = key_at(i);
      if ((k & above) == prefix) atomicAdd(&hist[(k >> shift) & mask], 1);
    }
    cl.sync();
    // the cluster's counts, bins taken from the top: thread t adds up the bins 2t and 2t + 1
    int c1 = 0, c0 = 0;
    const int b1 = kBins - 1 - 2 * tid, b0 = b1 - 1;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      if (c < C) {
        const int2 h = *reinterpret_cast<const int2*>(cl.map_shared_rank(hist, c) + b0);
        c1 += h.y;
        c0 += h.x;
      }
    }
    int x = c1 + c0;
    const int own = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    if (warp == 0) {
      int y = warp_sum[lane];
      const int o0 = y;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
      }
      warp_sum[lane] = y - o0;
    }
    __syncthreads();
    const int64_t before = warp_sum[warp] + x - own;  // keys in higher bins
    if (want > before && want <= before + c1) {
      found_bin = b1;
      found_above = (int)before;
    } else if (want > before + c1 && want <= before + own) {
      found_bin = b0;
      found_above = (int)before + c1;
    }
    __syncthreads();
    prefix |= (uint32_t)found_bin << shift;
    want -= found_above;
    __syncthreads();
  }
  // prefix is the K-th largest key; the first `want` tokens that have it stay
  const int run = (m + kSelWarps - 1) / kSelWarps;
  const int i0 = min(m, warp * run), i1 = min(m, i0 + run);
  int eq = 0;
  for (int i = i0; i < i1; i += 32) {
    const bool is = i + lane < i1 && key_at(i + lane) == prefix;
    eq += __popc(__ballot_sync(0xffffffffu, is));
  }
  const int eq0 = (int)cluster_scan(cl, warp_box, &cta_box[0], (uint64_t)eq);
  const unsigned below = (1u << lane) - 1;
  // of a run of 32 tokens: which stay (eq_seen counts the equal ones before it)
  auto stays = [&](int i, int& eq_seen) {
    const uint32_t k = i + lane < i1 ? key_at(i + lane) : 0u;
    const bool is = i + lane < i1 && k == prefix;
    const unsigned e = __ballot_sync(0xffffffffu, is);
    const bool keep = i + lane < i1 && (k > prefix || (is && eq_seen + __popc(e & below) < want));
    eq_seen += __popc(e);
    return keep;
  };
  int movers = 0, holes = 0, seen = eq0;
  for (int i = i0; i < i1; i += 32) {
    const bool keep = stays(i, seen);
    const int64_t t = lo + i + lane;
    movers += __popc(__ballot_sync(0xffffffffu, keep && t >= K));
    holes += __popc(__ballot_sync(0xffffffffu, i + lane < i1 && !keep && t < K));
  }
  const uint64_t at = cluster_scan(cl, warp_box, &cta_box[1], (uint64_t)movers << 32 | (uint32_t)holes);
  int mv = (int)(at >> 32), ho = (int)(uint32_t)at;
  seen = eq0;
  for (int i = i0; i < i1; i += 32) {
    const bool keep = stays(i, seen);
    const int64_t t = lo + i + lane;
    const bool mover = keep && t >= K, hole = i + lane < i1 && !keep && t < K;
    const unsigned bm = __ballot_sync(0xffffffffu, mover), bh = __ballot_sync(0xffffffffu, hole);
    if (mover) a.src[r * a.move_cols + mv + __popc(bm & below)] = (int)t;
    if (hole) a.dst[r * a.move_cols + ho + __popc(bh & below)] = (int)t;
    if (keep && t < K) {
      a.new_w[r * a.new_sr + t] = __ldg(a.w + r * a.w_sr + t);
      a.new_p[r * a.new_sr + t] = __ldg(a.pos + r * a.pos_sr + t);
    }
    mv += __popc(bm);
    ho += __popc(bh);
  }
  // the last warp of the last CTA has counted all movers
  if (rank == C - 1 && warp == kSelWarps - 1 && lane == 0) a.count[r] = mv;
  cl.sync();  // no CTA leaves while a peer may still read its sums
}

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 4;  // rows a warp moves together, their loads all in flight

// Moves the listed rows, their weights and positions.  A warp takes kMoveRows moves of a request
// at a time; blocks of a request stride over its list.
// 83 us for the 16 requests' kept rows past the budget of 12,288 (2 KB rows read and written once).
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a) {
  const int r = blockIdx.y, lane = threadIdx.x & 31;
  const int count = __ldg(a.count + r);
  const int warps = gridDim.x * (kMoveThreads / 32);
  for (int i0 = (blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5)) * kMoveRows; i0 < count; i0 += warps * kMoveRows) {
    // lanes 0 .. kMoveRows - 1 resolve one move each
    int64_t from = -1, to = -1;
    if (lane < kMoveRows && i0 + lane < count) {
      const int s = a.src[r * a.move_cols + i0 + lane], d = a.dst[r * a.move_cols + i0 + lane];
      const int ps = __ldg(a.bt + r * a.bt_stride + s / a.page_size), pd = __ldg(a.bt + r * a.bt_stride + d / a.page_size);
      a.new_w[r * a.new_sr + d] = __ldg(a.w + r * a.w_sr + s);
      a.new_p[r * a.new_sr + d] = __ldg(a.pos + r * a.pos_sr + s);
      if (ps >= 0 && ps < a.num_pages && pd >= 0 && pd < a.num_pages) {  // else there is no row to move
        from = (int64_t)ps * a.page_b + s % a.page_size * a.tok_b;
        to = (int64_t)pd * a.page_b + d % a.page_size * a.tok_b;
      }
    }
    int64_t f[kMoveRows], d[kMoveRows];
#pragma unroll
    for (int k = 0; k < kMoveRows; ++k) {
      f[k] = __shfl_sync(0xffffffffu, from, k);
      d[k] = __shfl_sync(0xffffffffu, to, k);
    }
    if (a.vec) {
      for (int64_t c = lane * 16; c < a.row_b; c += 32 * 16) {
        uint4 v[kMoveRows];
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k)
          if (f[k] >= 0) v[k] = __ldcs(reinterpret_cast<const uint4*>(a.cache + f[k] + c));
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k)
          if (f[k] >= 0) *reinterpret_cast<uint4*>(a.cache + d[k] + c) = v[k];
      }
    } else {
      for (int k = 0; k < kMoveRows; ++k)
        if (f[k] >= 0)
          for (int64_t c = lane; c < a.row_b; c += 32) a.cache[d[k] + c] = a.cache[f[k] + c];
    }
  }
}

struct EvictPlan {
  int64_t move_cols, ws_src, ws_dst, ws_count, ws_total;
};

int make_evict_plan(const qmla_evict_params* p, EvictPlan* pl) {
  if (!p || p->num_reqs < 0 || p->budget < 0 || p->cols < 0 || p->page_size <= 0 || p->kv_num_pages < 0 ||
      p->block_table_cols < 0 || p->row_bytes <= 0 || p->new_cols < std::min<int64_t>(p->budget, p->cols) ||
      p->token_stride_bytes < p->row_bytes)
    return QMLA_E_INVALID;
  if (p->cols > INT32_MAX / 2 || p->num_reqs > 65535) return QMLA_E_UNSUPPORTED;
  // a move fills a place below K with a token at or above it
  pl->move_cols = std::min<int64_t>(p->budget, p->cols);
  int64_t w = 0;
  pl->ws_src = w;
  w = align_up(w + 4 * pl->move_cols * p->num_reqs, 256);
  pl->ws_dst = w;
  w = align_up(w + 4 * pl->move_cols * p->num_reqs, 256);
  pl->ws_count = w;
  w = align_up(w + 4 * (int64_t)p->num_reqs, 256);
  pl->ws_total = w;
  return QMLA_OK;
}

}  // namespace

extern "C" {

int qmla_evict_workspace_bytes(const qmla_evict_params* p, int64_t* bytes) try {
  if (!bytes) return QMLA_E_INVALID;
  EvictPlan pl;
  const int rc = make_evict_plan(p, &pl);
  if (rc != QMLA_OK) return rc;
  *bytes = pl.ws_total;
  return QMLA_OK;
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

int qmla_evict(const qmla_evict_params* p, void* stream) try {
  EvictPlan pl;
  const int rc = make_evict_plan(p, &pl);
  if (rc != QMLA_OK) return rc;
  if (p->num_reqs == 0) return QMLA_OK;
  if ((p->cols > 0 && (!p->weights || !p->positions)) || (p->new_cols > 0 && (!p->new_weights || !p->new_positions)) ||
      !p->seq_lens || !p->new_lens || !p->kv_cache || !p->block_table)
    return QMLA_E_INVALID;
  if (!p->workspace || p->workspace_bytes < pl.ws_total) return QMLA_E_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0) return QMLA_E_ALIGNMENT;
  const DevInfo di = dev_info(p->device);
  if (!di.ok) return QMLA_E_CUDA;
  DeviceGuard dg(p->device);
  if (!dg.ok()) return QMLA_E_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  uint8_t* ws = reinterpret_cast<uint8_t*>(p->workspace);
  EvictArgs a;
  memset(&a, 0, sizeof(a));
  a.w = p->weights;
  a.w_sr = p->weights_stride_req;
  a.pos = p->positions;
  a.pos_sr = p->positions_stride_req;
  a.cols = p->cols;
  a.lens = p->seq_lens;
  a.budgets = p->budgets;
  a.budget = p->budget;
  a.sinks = p->sinks;
  a.recent_from = p->recent_from;
  a.new_w = p->new_weights;
  a.new_p = p->new_positions;
  a.new_sr = p->new_stride_req;
  a.new_cols = p->new_cols;
  a.new_lens = p->new_lens;
  a.src = reinterpret_cast<int32_t*>(ws + pl.ws_src);
  a.dst = reinterpret_cast<int32_t*>(ws + pl.ws_dst);
  a.count = reinterpret_cast<int32_t*>(ws + pl.ws_count);
  a.move_cols = pl.move_cols;
  a.reqs = p->num_reqs;
  a.cache = reinterpret_cast<uint8_t*>(p->kv_cache);
  a.page_b = p->page_stride_bytes;
  a.tok_b = p->token_stride_bytes;
  a.num_pages = p->kv_num_pages;
  a.row_b = p->row_bytes;
  a.bt = p->block_table;
  a.bt_stride = p->block_table_stride;
  a.bt_cols = p->block_table_cols;
  a.page_size = p->page_size;
  a.vec = reinterpret_cast<uintptr_t>(a.cache) % 16 == 0 && a.page_b % 16 == 0 && a.tok_b % 16 == 0 && a.row_b % 16 == 0;
  // CTAs of a request: one for every 8192 columns
  int C = 1;
  while (C < kMaxCluster && (int64_t)C * 8192 < p->cols) C *= 2;
  const int64_t per_cta = p->cols / C + 1;
  a.keys_fit = per_cta <= kMaxKeys;
  const size_t smem = a.keys_fit ? (size_t)per_cta * 4 : 0;
  if (!allow_smem(evict_select_kernel, kMaxKeys * 4)) return QMLA_E_CUDA;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)p->num_reqs * C);
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, evict_select_kernel, (const EvictArgs)a) != cudaSuccess) return QMLA_E_CUDA;
  if (pl.move_cols > 0) {
    // 8 blocks per SM between the requests, no more than the longest list needs
    const int64_t most = (pl.move_cols + kMoveRows * (kMoveThreads / 32) - 1) / (kMoveRows * (kMoveThreads / 32));
    const int64_t share = std::max<int64_t>(1, (8 * (int64_t)di.sms + p->num_reqs - 1) / p->num_reqs);
    evict_move_kernel<<<dim3((unsigned)std::min(most, share), p->num_reqs), kMoveThreads, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? QMLA_OK : QMLA_E_CUDA;
} catch (...) {  // no exception leaves a C entry
  return QMLA_E_CUDA;
}

}  // extern "C"
