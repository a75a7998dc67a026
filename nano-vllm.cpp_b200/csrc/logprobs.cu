// logprobs.cu -- per logits row: the log-probability and rank of a given
// token, the row's entropy and its top alternatives.
//
//   m = max x,  S = sum e^(x - m),  T = sum e^(x - m) (x - m)
//   log p_i = x_i - m - log S,  H = log S - T / S
//   rank of t: the number of ids before it in the order (value descending,
//   id ascending); the top k are the first k ids of that order
//
// H is written with x - m, not x: log S - T / S then has no cancellation of
// large terms.  Sums are f32 (a lane's 32 terms of a tile, then a running sum
// per lane, then a tree), rescaled when a tile raises the maximum.
//
// One pass over the logits, bound by memory: a warp takes tiles of 1,024
// logits (32 per lane, all loads of a tile in flight), about ten instructions
// per logit.  The top k cost the pass nothing but the tiles' maxima, which the
// running maximum needs anyway: an id of the top k lies in one of the k tiles
// whose maxima come first (each of those k tiles holds at least one id that
// precedes every id of any other tile), so the finish ranks the maxima,
// rereads k tiles (from L2) and ranks the few logits that reach the k-th
// maximum.  With fewer than k tiles, or more such logits than kMaxCandidates (sorted
// logits), that limit is the k-th largest of kThreads interleaved subsets'
// maxima; what is still too many (ties) is taken one after another.
//
// Measured: 256 rows of 151,936 f32 logits, top 5, 34.9 us (4.5 TB/s of logits,
// 69 % of the measured copy rate; the finish of the last rows is what the
// loads do not cover); one bf16 row, top 20, 10.6 us (the chain of a tile or
// two per warp, the cluster's hand-over and the finish).
//
// A row is one cluster of 1 to 8 CTAs, more where there are fewer rows
// (launch_token_logprobs); the CTAs hand their sums and tile maxima to CTA 0
// through distributed shared memory, so there is no workspace, no second
// launch, and nothing that depends on the order of arrival.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "internal.h"

namespace nvattn {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 1024;
constexpr int kMaxTiles = kLogprobsMaxVocab / kTile;
constexpr int kMaxCluster = 8;
constexpr int kMaxCandidates = 1024;
static_assert(kMaxTop <= kThreads, "subsets");
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  int n_vocab, top_k;
  int row0;  // the launch's first row of the call
  long long row_stride;
  const void* logits;
  const int32_t* tokens;
  float* logprobs;
  float* entropy;
  int32_t* ranks;
  int32_t* top_ids;
  float* top_logprobs;
  DeviceStatus* status;
};

struct Sums {
  float m, s, t;
  int before;  // ids before the given token
};

struct Smem {
  alignas(16) uint32_t tile_key[kMaxTiles];  // CTA 0: every tile's maximum, as an ordered key
  Sums part[kMaxCluster];        // CTA 0: the CTAs' sums
  Sums warp[kWarps];
  int tile[kMaxTop];             // the chosen tiles
  int id[kMaxCandidates];
  alignas(16) uint64_t order[kMaxCandidates];
  uint64_t best[kWarps];
  uint32_t floor_key;
  int count;
  float m, log_s;
};

// The order of logits: larger first; a NaN counts as -infinity, -0 as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr uint32_t kMinusInfinity = 0x007fffffu;  // ordered(-infinity), the least key
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// How many of the n keys (n rounded up to a multiple of 4 and zero there) come
// before `mine` at place i: larger ones, and equal ones at a lower place.
__device__ __forceinline__ int rank_of(const uint32_t* keys, int n, uint32_t mine, int i) {
  int rank = 0;
#pragma unroll 4
  for (int j = 0; j < n; j += 4) {
    const uint4 o = *reinterpret_cast<const uint4*>(keys + j);
    rank += (o.x > mine || (o.x == mine && j < i)) + (o.y > mine || (o.y == mine && j + 1 < i)) +
            (o.z > mine || (o.z == mine && j + 2 < i)) +
            (o.w > mine || (o.w == mine && j + 3 < i));
  }
  return rank;
}

template <bool kBf16>
__device__ __forceinline__ float load1(const Args& a, const void* row, int i) {
  if constexpr (kBf16)
    return __uint_as_float((uint32_t)static_cast<const uint16_t*>(row)[i] << 16);
  else
    return static_cast<const float*>(row)[i];
}

// The id of a lane's e-th logit of a tile (kVec: 16-byte loads).
template <bool kBf16, bool kVec>
__device__ __forceinline__ int id_of(int tile, int lane, int e) {
  constexpr int kPer = kBf16 ? 8 : 4;
  return tile * kTile +
         (kVec ? (e / kPer) * (32 * kPer) + lane * kPer + e % kPer : e * 32 + lane);
}

// A lane's 32 logits of a tile; -infinity behind the vocabulary.
template <bool kBf16, bool kVec>
__device__ __forceinline__ void load_tile(const Args& a, const void* row, int tile, int lane,
                                          float (&x)[32]) {
  const bool whole = (tile + 1) * kTile <= a.n_vocab;
  if (kVec && whole) {
    if constexpr (kBf16) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(
            static_cast<const uint16_t*>(row) + id_of<kBf16, kVec>(tile, lane, 8 * j)));
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[8 * j + 2 * e] = bf16lo_to_f32(u[e]);
          x[8 * j + 2 * e + 1] = bf16hi_to_f32(u[e]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(
            static_cast<const float*>(row) + id_of<kBf16, kVec>(tile, lane, 4 * j)));
        x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const int i = id_of<kBf16, kVec>(tile, lane, e);
      x[e] = i < a.n_vocab ? load1<kBf16>(a, row, i) : -INFINITY;
    }
  }
}

// Sums under a new reference (m_new >= a.m; -infinity: nothing summed yet).
// The step between them counts as -1e4 at most, where its factor is 0 already:
// from a tile masked with the type's lowest value it would overflow beside s,
// and 0 * -infinity is NaN.
__device__ __forceinline__ void rescale(float m, float m_new, float& s, float& t) {
  if (m_new == m || m == -INFINITY) return;
  const float d = fmaxf(m - m_new, -1.0e4f);
  const float f = fast_exp2(d * kLog2e);
  t = f * fmaf(d, s, t);
  s *= f;
}

__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  rescale(a.m, m, a.s, a.t);
  rescale(b.m, m, b.s, b.t);
  return {m, a.s + b.s, a.t + b.t, a.before + b.before};
}

template <bool kBf16, bool kVec>
__global__ void __launch_bounds__(kThreads, 2) token_logprobs_kernel(Args a) {
  __shared__ Smem sm;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = (int)cluster_ctarank(), n_ctas = (int)gridDim.x, row_i = blockIdx.y;
  const void* row = kBf16 ? static_cast<const void*>(static_cast<const uint16_t*>(a.logits) +
                                                     row_i * a.row_stride)
                          : static_cast<const float*>(a.logits) + row_i * a.row_stride;
  const int n_tiles = (a.n_vocab + kTile - 1) / kTile;

  const int token = a.tokens != nullptr ? a.tokens[row_i] : -1;
  const bool has_token = token >= 0 && token < a.n_vocab;
  float raw_xt = __uint_as_float(0x7fc00000u), xt = INFINITY;  // the token's logit; NaN as -inf
  const uint32_t keys0 = smem_peer(sm.tile_key, 0);
  if (n_ctas > 1) cluster_sync();  // CTA 0 has started: its shared memory may be written

  // ---- the pass ----
  Sums r = {-INFINITY, 0.0f, 0.0f, 0};
  const int tile0 = cta * kWarps + warp;
  for (int tile = tile0; tile < n_tiles || tile == tile0; tile += n_ctas * kWarps) {
    float x[32];
    if (tile < n_tiles) load_tile<kBf16, kVec>(a, row, tile, lane, x);
    if (tile == tile0 && has_token) {
      // behind the first tile's loads, which do not wait for the token
      raw_xt = load1<kBf16>(a, row, token);
      xt = fmaxf(raw_xt, -INFINITY);
    }
    if (tile >= n_tiles) break;
    float top = x[0];
#pragma unroll
    for (int e = 1; e + 1 < 32; e += 2) top = fmax3(top, x[e], x[e + 1]);
    top = fmaxf(fmaxf(top, x[31]), -INFINITY);
    const uint32_t key = __reduce_max_sync(0xffffffffu, ordered(top));
    if (lane == 0 && a.top_k > 0) st_cluster_u32(keys0 + 4 * tile, key);
    const float m = fmaxf(r.m, value_of(key));
    rescale(r.m, m, r.s, r.t);
    r.m = m;
    const float ref = m == -INFINITY ? 0.0f : m;
    float s[4] = {0, 0, 0, 0}, t[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const float z = x[e] - ref;
      const float p = fast_exp2(z * kLog2e);
      s[e & 3] += p;
      t[e & 3] = fmaf(p, fmaxf(z, -1.0e4f), t[e & 3]);  // 0 * -inf counts as 0
    }
    r.s += (s[0] + s[1]) + (s[2] + s[3]);
    r.t += (t[0] + t[1]) + (t[2] + t[3]);
    // (a tile whose maximum lies below the token's logit has nothing before it:
    // most tiles, where the token is a likely one)
    if (has_token && value_of(key) >= xt) {
      int n = 0;
      if (token >= (tile + 1) * kTile) {  // equals come before the token
#pragma unroll
        for (int e = 0; e < 32; ++e) n += fmaxf(x[e], -INFINITY) >= xt;
      } else if (token < tile * kTile) {
#pragma unroll
        for (int e = 0; e < 32; ++e) n += x[e] > xt;
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float v = fmaxf(x[e], -INFINITY);
          n += v > xt || (v == xt && id_of<kBf16, kVec>(tile, lane, e) < token);
        }
      }
      r.before += n;
    }
  }

  // ---- the warp's, the CTA's, the row's sums ----
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
    r.t += __shfl_xor_sync(0xffffffffu, r.t, o);
  }
  r.before = __reduce_add_sync(0xffffffffu, r.before);
  if (lane == 0) sm.warp[warp] = r;
  __syncthreads();
  if (warp == 0) {
    Sums w = lane < kWarps ? sm.warp[lane] : Sums{-INFINITY, 0.0f, 0.0f, 0};
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const Sums other = {__shfl_xor_sync(0xffffffffu, w.m, o),
                          __shfl_xor_sync(0xffffffffu, w.s, o),
                          __shfl_xor_sync(0xffffffffu, w.t, o),
                          __shfl_xor_sync(0xffffffffu, w.before, o)};
      w = (lane & o) ? join(other, w) : join(w, other);
    }
    if (lane == 0) {
      const uint32_t dst = smem_peer(&sm.part[cta], 0);
      st_cluster_u32(dst, __float_as_uint(w.m));
      st_cluster_u32(dst + 4, __float_as_uint(w.s));
      st_cluster_u32(dst + 8, __float_as_uint(w.t));
      st_cluster_u32(dst + 12, (uint32_t)w.before);
    }
  }
  cluster_sync();
  if (cta != 0) return;

  // ---- the k tiles that hold the top k; beside it, one thread (of the last
  // warp, which ranks no tile unless there are many) the row's values ----
  const int k_tiles = min(a.top_k, n_tiles);
  if (threadIdx.x == 0) {
    sm.count = 0;
    sm.floor_key = 0;
  }
  for (int i = n_tiles + threadIdx.x; i < (n_tiles + 3) / 4 * 4; i += kThreads)
    sm.tile_key[i] = 0;  // precedes nothing
  __syncthreads();
  if (threadIdx.x == kThreads - 1) {
    Sums w = sm.part[0];
    for (int i = 1; i < n_ctas; ++i) w = join(w, sm.part[i]);
    const float m = w.m == -INFINITY ? 0.0f : w.m;
    const float log_s = logf(w.s);
    sm.m = m;
    sm.log_s = log_s;
    if (a.entropy != nullptr) a.entropy[row_i] = log_s - w.t / w.s;
    if (a.tokens != nullptr) {
      if (!has_token) record_error(a.status, NVATTN_ERR_OUT_OF_RANGE, 95, a.row0 + row_i);
      if (a.logprobs != nullptr) a.logprobs[row_i] = raw_xt - m - log_s;
      if (a.ranks != nullptr) a.ranks[row_i] = has_token ? w.before : -1;
    }
  }
  if (a.top_k <= 0) return;
  for (int i = threadIdx.x; i < n_tiles; i += kThreads) {
    const uint32_t mine = sm.tile_key[i];
    const int rank = rank_of(sm.tile_key, n_tiles, mine, i);
    if (rank < k_tiles) {
      sm.tile[rank] = i;
      if (rank == a.top_k - 1) sm.floor_key = mine;
    }
  }
  __syncthreads();

  // ---- their logits that reach a limit which k of them reach ----
  // A warp rereads a tile at a time, 32 logits per lane.  (This part runs once
  // per row and is kept short: its instructions come from memory.)
  int n = kMaxCandidates + 1;
  for (int attempt = n_tiles >= a.top_k ? 0 : 1; attempt < 2 && n > kMaxCandidates; ++attempt) {
    if (attempt == 1) {
      float top = -INFINITY;
#pragma unroll 1
      for (int i = warp; i < k_tiles; i += kWarps) {
        float x[32];
        load_tile<kBf16, kVec>(a, row, sm.tile[i], lane, x);
#pragma unroll
        for (int e = 0; e < 32; e += 2) top = fmax3(top, x[e], x[e + 1]);
      }
      // the k-th largest of the threads' maxima, bit by bit
      const uint32_t mine = ordered(top);
      uint32_t kth = 0;
#pragma unroll 1
      for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1)
        if (__syncthreads_count(mine >= (kth | bit)) >= a.top_k) kth |= bit;
      if (threadIdx.x == 0) {
        sm.floor_key = kth;
        sm.count = 0;
      }
      __syncthreads();
    }
    const float floor = sm.floor_key > kMinusInfinity ? value_of(sm.floor_key) : -INFINITY;
#pragma unroll 1
    for (int i = warp; i < k_tiles; i += kWarps) {
      const int tile = sm.tile[i];
      uint32_t reach = 0;
      {
        float x[32];
        load_tile<kBf16, kVec>(a, row, tile, lane, x);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          reach |= (fmaxf(x[e], -INFINITY) >= floor ? 1u : 0u) << e;
      }
#pragma unroll 1
      for (; reach != 0; reach &= reach - 1) {
        const int id = id_of<kBf16, kVec>(tile, lane, __ffs(reach) - 1);
        if (id < a.n_vocab) {
          const int at = atomicAdd(&sm.count, 1);
          if (at < kMaxCandidates) sm.id[at] = id;
        }
      }
    }
    __syncthreads();
    n = sm.count;
    __syncthreads();
  }
  const long long out = (long long)row_i * a.top_k;
  if (n <= kMaxCandidates) {
    // (key, ~id) as one 64-bit number is the order, largest first
    for (int i = threadIdx.x; i < (n + 1) / 2 * 2; i += kThreads)
      sm.order[i] = i < n ? (uint64_t)ordered(load1<kBf16>(a, row, sm.id[i])) << 32 |
                                (uint32_t)~sm.id[i]
                          : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t mine = sm.order[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; j += 2) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sm.order[j]);
        rank += (o.x > mine) + (o.y > mine);
      }
      if (rank < a.top_k) {
        a.top_ids[out + rank] = (int)~(uint32_t)mine;
        a.top_logprobs[out + rank] = value_of((uint32_t)(mine >> 32)) - sm.m - sm.log_s;
      }
    }
    return;
  }
  // Too many to rank at once: the first, then the first after it, and so on.
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t best = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < k_tiles * kTile; i += kThreads) {
      const int id = sm.tile[i / kTile] * kTile + i % kTile;
      if (id < a.n_vocab) {
        const uint64_t v = (uint64_t)ordered(load1<kBf16>(a, row, id)) << 32 | (uint32_t)~id;
        if (v < last && v > best) best = v;
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
      best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)best, o));
    if (lane == 0) sm.best[warp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) best = max(best, sm.best[w]);
    last = best;
    if (threadIdx.x == 0) {
      const int id = (int)~(uint32_t)best;
      a.top_ids[out + k] = id;
      a.top_logprobs[out + k] = value_of((uint32_t)(best >> 32)) - sm.m - sm.log_s;
    }
    __syncthreads();  // sm.best is free
  }
}

}  // namespace

nvattn_status launch_token_logprobs(nvattn_handle* h, int n_rows, int n_vocab, const void* logits,
                                    nvattn_dtype dtype, long long row_stride,
                                    const int32_t* tokens, float* logprobs, float* entropy,
                                    int32_t* ranks, int top_k, int32_t* top_ids,
                                    float* top_logprobs, cudaStream_t stream) {
  if (n_rows == 0) return NVATTN_OK;
  Args a = {};
  a.n_vocab = n_vocab;
  a.top_k = top_k;
  a.row_stride = row_stride;
  a.logits = logits;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.ranks = ranks;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.status = h->status_dev;
  const bool bf16 = dtype == NVATTN_DTYPE_BF16;
  const int el = bf16 ? 2 : 4;
  const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 && row_stride * el % 16 == 0;
  // CTAs per row: as many as leave every warp a tile, while all rows stay
  // resident (two CTAs per SM).  More CTAs per row than that only add waits
  // for CTA 0's finish: 256 rows of 151,936 f32 took 35.5 us with one CTA per
  // row, 45 with two, 54 with four, 75 with eight.
  const int n_tiles = (n_vocab + kTile - 1) / kTile;
  int cluster = 1;
  while (cluster < kMaxCluster && cluster * kWarps < n_tiles &&
         2LL * cluster * n_rows <= 2LL * h->sm_count)
    cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto kernel = bf16 ? (vec ? token_logprobs_kernel<true, true> : token_logprobs_kernel<true, false>)
                     : (vec ? token_logprobs_kernel<false, true>
                            : token_logprobs_kernel<false, false>);
  constexpr int kMaxRowsPerLaunch = 65535;  // the grid's y extent
  for (int r0 = 0; r0 < n_rows; r0 += kMaxRowsPerLaunch) {
    const int n = std::min(n_rows - r0, kMaxRowsPerLaunch);
    cfg.gridDim = dim3(cluster, n);
    a.row0 = r0;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return NVATTN_ERR_CUDA;
    a.logits = static_cast<const char*>(a.logits) + (long long)n * row_stride * el;
    if (a.tokens) a.tokens += n;
    if (a.logprobs) a.logprobs += n;
    if (a.entropy) a.entropy += n;
    if (a.ranks) a.ranks += n;
    if (a.top_ids) a.top_ids += (long long)n * top_k;
    if (a.top_logprobs) a.top_logprobs += (long long)n * top_k;
  }
  return cudaGetLastError() == cudaSuccess ? NVATTN_OK : NVATTN_ERR_CUDA;
}

}  // namespace nvattn
