// tree_decode.cu -- paged attention for trees of drafted tokens over the BF16
// cache, on the tcgen05 tensor cores (sm_100a).
//
// Sequence s brings N_s nodes, the last N_s positions of its context; node i
// attends every key before them and those nodes j whose bit is set in its
// mask:  o_i = sum_t softmax_t(scale q_i.k_t) v_t  over those t.
//
// A unit is (sequence, kv head, tile of 128 query rows); row r of a unit's
// sequence is node r / G, query head r % G.  So all nodes and all query heads
// of a kv head read its keys together: 512 bytes per token and kv head for up
// to 128 rows, bound by memory until a kv head has several row tiles (whose
// keys then come from L2).  The units' 64-key tiles are split evenly over one
// CTA per SM (tile_split.cuh); the partials that this makes are merged by the
// CTA that finishes a unit last, in CTA order.
//
//   warp 0      TMA producer: K and V tiles of 16 KiB (two boxes of 64 dims x
//               64 tokens, 128-byte swizzle) through a ring of kSlots that
//               runs on across units.
//   warp 1      TMEM allocation; one lane issues the MMAs (M = 128 rows):
//                 S(j) = Q K^T   N = 64 keys, A = Q from TMEM
//                 O   += P V     N = 128 dims, K = 64 keys, A = P from TMEM
//               S(j+1) before P V(j), so that the softmax never waits for the
//               tensor cores; both A operands come from TMEM, which leaves the
//               shared-memory reads to K and V.
//   warps 2-5   thread = row = TMEM lane: queries into TMEM, mask, online
//               softmax in the log2 domain with lazy rescaling of O, P over
//               the columns of its own S, epilogue.
// Precision: products of bf16 operands, f32 sums.  bf16 queries are one
// operand and P is a sum of two bf16 terms (16 bits; one term, 8 bits, would
// add as much error as the rounding of a bf16 output itself).  f32 queries and
// their P are sums of three bf16 terms, 24 bits: f32 in, f32 out.
// TMEM columns: Q [0, 64 kQ), O [192, 320), then two S / P buffers of 96.
#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "tile_split.cuh"

namespace nvattn {
namespace {

constexpr int kD = 128;
constexpr int kRows = 128;
constexpr int kTile = 64;  // keys per tile
constexpr int kThreads = 6 * 32;
constexpr int kSlots = 13;
constexpr int kHalfBytes = kTile * 64 * 2;  // one box: 64 tokens x 64 dims
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 192, kColS = 320, kColsS = 96;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;  // log2: rescale O only when a row's maximum grows past 2^8
// A unit's start and end cost about as much as this many tiles (its queries
// into TMEM, the first S and the epilogue do not overlap its neighbours').
constexpr int kUnitCost = 4;

struct TreeParams {
  int Hq, Hkv, G, layer, block_size, max_blocks, n_seqs, n_nodes, max_nodes, mask_words;
  int max_context;
  long long n_slots, num_blocks;
  float scale_log2;
  const void* q;
  const int32_t* cu_nodes;
  const uint64_t* mask;
  const int32_t* block_tables;
  const int32_t* context_lens;
  void* out;
  float* part;   // [CTA][2][kTreePartFloats]: O [dim][row], references, sums
  int* tickets;  // [CTA], zero between launches
  DeviceStatus* status;
};

struct __align__(1024) TreeSmem {
  uint16_t kv[kSlots][2][kTile * 64];  // [slot][d half][token][64]
  uint64_t full[kSlots], empty[kSlots];
  uint64_t q_ready, s_full[2], p_full[2], o_done[2];
  uint32_t bad[2][2];  // [tile & 1]: keys of the tile whose V row holds a NaN or an infinity
  uint32_t tmem_base;
  int abort_flag;
  int skip;
  int last;
};
static_assert(sizeof(TreeSmem) + 1024 <= 227 * 1024, "shared memory");

__device__ __forceinline__ int ring_slot(int idx) { return idx % kSlots; }
__device__ __forceinline__ uint32_t ring_parity(int idx) { return (uint32_t)(idx / kSlots) & 1u; }

// A sequence's nodes and context; n = 0 where it has none or its metadata is
// unusable (`report`: recorded then).
struct SeqInfo {
  int node0, n, ctx;
};
__device__ __forceinline__ SeqInfo seq_info(const TreeParams& p, int s, bool report) {
  const int a = p.cu_nodes[s], b = p.cu_nodes[s + 1];
  int ctx = p.context_lens[s];
  if (a < 0 || b < a || b > p.n_nodes || b - a > p.max_nodes) {
    if (report) record_error(p.status, NVATTN_ERR_OUT_OF_RANGE, 100, b);
    return {0, 0, 0};
  }
  if (ctx < b - a || ctx > p.max_context) {  // the nodes are part of the context
    if (report) record_error(p.status, NVATTN_ERR_OUT_OF_RANGE, 101, ctx);
    return {0, 0, 0};
  }
  return {a, b - a, ctx};
}
__device__ __forceinline__ int row_tiles(const TreeParams& p, int n) {
  return (n * p.G + kRows - 1) / kRows;
}
__device__ __forceinline__ int key_tiles(int ctx) { return (ctx + kTile - 1) / kTile; }

// One unit's part of the CTA's run: key tiles [j0, j1).
struct Segment {
  int seq, head, row_tile, j0, j1, n_tiles;
  SeqInfo info;
  long long unit0;  // place of the unit's first tile
};

// Walks the segments of a run; every role walks the same ones.
struct Walker {
  long long at, end, per;
  int seq, unit;  // the unit that `at` lies in
  SeqInfo info;

  __device__ __forceinline__ void start(const TreeParams& p, const tilesplit::Run& r) {
    at = r.begin;
    end = r.end;
    per = r.per;
    seq = r.seq;
    unit = 0;
    if (at >= end) return;
    info = seq_info(p, seq, false);
    const int span = key_tiles(info.ctx) + kUnitCost;
    unit = (int)((at - r.seq_first) / span);
    offset = (int)((at - r.seq_first) % span);
  }
  int offset;  // place of `at` in its unit

  __device__ __forceinline__ bool next(const TreeParams& p, Segment& s) {
    while (at < end) {
      const int tiles = key_tiles(info.ctx);
      const int left = tiles + kUnitCost - offset;
      const int take = (int)min((long long)left, end - at);
      const int j0 = max(offset - kUnitCost, 0), j1 = offset + take - kUnitCost;
      bool some = j1 > j0;
      if (some) {
        const int rt = row_tiles(p, info.n);
        s = {seq, unit / rt, unit % rt, j0, j1, tiles, info, at - offset + kUnitCost};
      }
      at += take;
      offset = 0;
      if (take == left && at < end) {
        if (++unit == p.Hkv * row_tiles(p, info.n)) {
          unit = 0;
          do info = seq_info(p, ++seq, false);
          while (info.n == 0);  // (`at` < end: a later sequence has places)
        }
      }
      if (some) return true;
    }
    return false;
  }
};

// The next bf16 term of two values; they keep what is left.
__device__ __forceinline__ void split_term(float& x0, float& x1, uint32_t& packed) {
  packed = cvt_bf16x2(x0, x1);
  x0 -= bf16lo_to_f32(packed);
  x1 -= bf16hi_to_f32(packed);
}

// kF32: f32 queries and outputs (three terms each), else bf16 (one and two).
template <bool kF32>
__global__ void __launch_bounds__(kThreads, 1)
    tree_decode_kernel(const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, TreeParams p) {
  constexpr int kQ = kF32 ? 3 : 1, kP = kF32 ? 3 : 2;
  static_assert(64 * kQ <= kColO && 32 * kP <= kColsS && kTile <= kColsS, "TMEM columns");
  extern __shared__ uint8_t smem_raw[];
  TreeSmem& sm = *reinterpret_cast<TreeSmem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.q_ready, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_done[i], 1);
      sm.bad[i][0] = sm.bad[i][1] = 0;
    }
    sm.abort_flag = 0;
    sm.skip = timeout_recorded(p.status);
    fence_barrier_init();
  }
  if (blockIdx.x == 0)  // every sequence's metadata is checked once
    for (int s = threadIdx.x; s < p.n_seqs; s += kThreads) seq_info(p, s, true);
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, kTmemCols);
    tmem_relinquish();
  }
  const tilesplit::Run run = tilesplit::find_run(p.n_seqs, blockIdx.x, gridDim.x, [&](int s) {
    const SeqInfo i = seq_info(p, s, false);
    return tilesplit::SeqTiles{p.Hkv * row_tiles(p, i.n), key_tiles(i.ctx) + kUnitCost};
  });
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_flag = &sm.abort_flag;
  Walker walk;
  walk.start(p, run);
  if (sm.skip) walk.at = walk.end;
  Segment seg;
  int g = 0;  // tiles of the run before the segment

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      const uint64_t policy = l2_policy_evict_first(), keep = l2_policy_evict_last();
      while (walk.next(p, seg)) {
        // keys that another row tile reads again stay in L2
        const uint64_t pol = row_tiles(p, seg.info.n) > 1 ? keep : policy;
        int block = -1;
        long long bid = 0;
        for (int j = seg.j0; j < seg.j1; ++j, ++g) {
          const int tok = j * kTile;
          if (tok / p.block_size != block) {
            block = tok / p.block_size;
            bid = p.block_tables[(long long)seg.seq * p.max_blocks + block];
            if (bid < 0 || bid >= p.num_blocks) {
              record_error(p.status, NVATTN_ERR_OUT_OF_RANGE, 102, bid);
              bid = 0;  // keep the pipeline flowing; the result is flagged invalid
            }
          }
          const int row = (int)((long long)p.layer * p.n_slots + bid * p.block_size +
                                tok % p.block_size);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int idx = 2 * g + kv, slot = ring_slot(idx);
            if (idx >= kSlots)
              mbar_wait(&sm.empty[slot], ring_parity(idx) ^ 1u, p.status, abort_flag, 103);
            const CUtensorMap* map = kv ? &tm_v : &tm_k;
            mbar_arrive_expect_tx(&sm.full[slot], 2 * kHalfBytes);
            tma_load_3d_hint(sm.kv[slot][0], map, &sm.full[slot], 0, seg.head, row, pol);
            tma_load_3d_hint(sm.kv[slot][1], map, &sm.full[slot], 64, seg.head, row, pol);
          }
        }
      }
      // Drain: the last load of every slot has landed before the CTA exits.
      for (int idx = max(0, 2 * g - kSlots); idx < 2 * g; ++idx)
        mbar_wait(&sm.full[ring_slot(idx)], ring_parity(idx), p.status, 104);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc_bf16_f32(kRows, kTile, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc_bf16_f32(kRows, kD, 0, 1);
      int n_seg = 0;
      while (walk.next(p, seg)) {
        mbar_wait(&sm.q_ready, n_seg & 1, p.status, abort_flag, 105);
        ++n_seg;
        const int n = seg.j1 - seg.j0;
        auto issue_s = [&](int gj) {
          const int slot = ring_slot(2 * gj);
          mbar_wait(&sm.full[slot], ring_parity(2 * gj), p.status, abort_flag, 106);
          tc_fence_after();
          const uint32_t d = tmem + kColS + (gj & 1) * kColsS;
#pragma unroll
          for (int t = kQ - 1; t >= 0; --t)  // the small terms first
#pragma unroll
            for (int k = 0; k < kD / 16; ++k)
              umma_bf16_ts(d, tmem + t * 64 + k * 8,
                           umma_desc_sw128(smem_u32(sm.kv[slot][k >> 2]) + (k & 3) * 32, 16, 1024),
                           idesc_s, (t < kQ - 1 || k > 0) ? 1u : 0u);
          umma_commit(&sm.s_full[gj & 1]);
          umma_commit(&sm.empty[slot]);
        };
        issue_s(g);
        for (int j = 0; j < n; ++j) {
          const int gj = g + j;
          if (j + 1 < n) issue_s(gj + 1);
          const int slot = ring_slot(2 * gj + 1);
          mbar_wait(&sm.p_full[gj & 1], (gj >> 1) & 1, p.status, abort_flag, 107);
          mbar_wait(&sm.full[slot], ring_parity(2 * gj + 1), p.status, abort_flag, 108);
          tc_fence_after();
          const uint32_t a = tmem + kColS + (gj & 1) * kColsS;
          const uint32_t v = smem_u32(sm.kv[slot][0]);
#pragma unroll
          for (int t = kP - 1; t >= 0; --t)
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k)
              umma_bf16_ts(tmem + kColO, a + t * 32 + k * 8,
                           umma_desc_sw128(v + (uint32_t)k * 16 * 128, kHalfBytes, 1024), idesc_o,
                           (j > 0 || t < kP - 1 || k > 0) ? 1u : 0u);
          umma_commit(&sm.o_done[gj & 1]);
          umma_commit(&sm.empty[slot]);
        }
        g += n;
      }
      // Drain: every MMA has completed before TMEM is released.
      if (g > 0) mbar_wait(&sm.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1, p.status, 109);
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int quad = warp & 3;  // TMEM lanes [32 * quad, 32 * quad + 32)
    const int r = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const int tid = (int)threadIdx.x - 64;
    while (walk.next(p, seg)) {
      const int n_rows = seg.info.n * p.G;
      const int row = seg.row_tile * kRows + r;
      const bool real = row < n_rows;
      const bool warp_real = seg.row_tile * kRows + quad * 32 < n_rows;
      const int node = seg.info.node0 + (real ? row / p.G : 0);
      const long long io =
          ((long long)node * p.Hq + (long long)seg.head * p.G + (real ? row % p.G : 0)) * kD;
      const int first = seg.info.ctx - seg.info.n;  // position of the sequence's first node
      // ---- queries into TMEM (the unit's S before are complete: they were
      // waited for by the softmax that read them) ----
      if (warp_real) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if constexpr (kF32) {
            float x[64];
            const float4* src =
                reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + io + 64 * hf);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float4 v = real ? src[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
            }
#pragma unroll
            for (int t = 0; t < kQ; ++t) {
              uint32_t w[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) split_term(x[2 * i], x[2 * i + 1], w[i]);
              tmem_st32(tmem + lane_off + t * 64 + hf * 32, w);
            }
          } else {
            uint32_t w[32];
            const uint4* src =
                reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + io + 64 * hf);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint4 v = real ? src[i] : make_uint4(0, 0, 0, 0);
              w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
            tmem_st32(tmem + lane_off + hf * 32, w);
          }
        }
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_ready);

      float m = -INFINITY, l = 0.0f;
      const int n = seg.j1 - seg.j0;
      for (int j = 0; j < n; ++j) {
        const int gj = g + j;
        const int col0 = (seg.j0 + j) * kTile;
        // Which of the tile's 64 keys the row attends.
        const bool special = col0 + kTile > first;  // holds nodes (or keys past the end)
        uint64_t allowed = ~0ull;
        if (special) {
          const int rel = col0 - first;  // the first key's place among the nodes
          uint64_t window = 0;
          if (real) {
            const uint64_t* words = p.mask + (long long)node * p.mask_words;
            if (rel < 0) {
              window = (words[0] << -rel) | ((1ull << -rel) - 1);
            } else {
              const int q = rel >> 6, sh = rel & 63;
              if (q < p.mask_words) window = words[q] >> sh;
              if (sh > 0 && q + 1 < p.mask_words) window |= words[q + 1] << (64 - sh);
            }
          }
          const int here = seg.info.ctx - col0;  // keys of the context from here on, >= 1
          allowed = here < kTile ? window & ((1ull << here) - 1) : window;
        }
        mbar_wait(&sm.s_full[gj & 1], (gj >> 1) & 1, p.status, abort_flag, 110);
        tc_fence_after();
        const uint32_t s_col = tmem + lane_off + kColS + (gj & 1) * kColsS;
        float x[64];
        if (warp_real) {
          uint32_t w[32];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            tmem_ld32(s_col + 32 * hf, w);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) x[32 * hf + i] = __uint_as_float(w[i]);
          }
        }
        if (special) {
          // V rows of nodes that hold a NaN or an infinity: 0 * NaN would
          // reach the rows whose masks leave the node out.  Such a row is
          // zeroed and noted, and makes the rows that attend it NaN.  Slots
          // past the context may hold anything and are zeroed.
          const int vidx = 2 * gj + 1, slot = ring_slot(vidx);
          mbar_wait(&sm.full[slot], ring_parity(vidx), p.status, abort_flag, 111);
          const int t = tid >> 1;  // token of the tile; two threads, a dim half each
          uint4* v = reinterpret_cast<uint4*>(
              reinterpret_cast<uint8_t*>(sm.kv[slot][tid & 1]) + t * 128);
          const bool past = col0 + t >= seg.info.ctx;
          bool bad = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 c = v[i];
            const uint32_t u[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              bad = bad || (u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u;
          }
          const uint32_t votes =
              __ballot_sync(0xffffffffu, bad && !past && col0 + t >= first);
          bad = (votes >> (lane & ~1)) & 3u;
          if (bad && (tid & 1) == 0) atomicOr(&sm.bad[gj & 1][t >> 5], 1u << (t & 31));
          if (bad || past) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          named_barrier_sync(1, 128);
          const uint64_t bad_keys = (uint64_t)sm.bad[gj & 1][1] << 32 | sm.bad[gj & 1][0];
          if (bad_keys & allowed) l = __uint_as_float(0x7fc00000u);
          named_barrier_sync(1, 128);
          // (set again two tiles on at the earliest, whose S follows this P)
          if (tid < 2) sm.bad[gj & 1][tid] = 0;
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = (allowed >> i) & 1 ? x[i] : -INFINITY;
        }
        if (warp_real) {
          float top = fmaxf(x[0], x[1]);
#pragma unroll
          for (int i = 2; i < 64; i += 2) top = fmax3(top, x[i], x[i + 1]);
          top *= p.scale_log2;
          const float m_new = top > m + kSlack ? top : m;
          const bool grows = m_new != m;
          if (__any_sync(0xffffffffu, grows)) {
            const float alpha = grows ? fast_exp2(m - m_new) : 1.0f;  // m = -inf: 0
            l *= alpha;
            m = m_new;
            if (j > 0) {
              // P V(j - 1) has finished: O is stable
              mbar_wait(&sm.o_done[(gj - 1) & 1], ((gj - 1) >> 1) & 1, p.status, abort_flag, 112);
              tc_fence_after();
              uint32_t w[32];
#pragma unroll
              for (int c = 0; c < kD; c += 32) {
                tmem_ld32(tmem + lane_off + kColO + c, w);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  w[i] = __float_as_uint(__uint_as_float(w[i]) * alpha);
                tmem_st32(tmem + lane_off + kColO + c, w);
              }
              tmem_wait_st();
            }
          }
          const float ref = m == -INFINITY ? 0.0f : m;  // a row without keys yet: weights 0
          float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            x[i] = fast_exp2(fmaf(x[i], p.scale_log2, -ref));
            s[i & 3] += x[i];
          }
          l += (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
          for (int t = 0; t < kP; ++t) {
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) split_term(x[2 * i], x[2 * i + 1], w[i]);
            tmem_st32(s_col + 32 * t, w);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[gj & 1]);
      }
      g += n;

      // ---- epilogue ----
      mbar_wait(&sm.o_done[(g - 1) & 1], ((g - 1) >> 1) & 1, p.status, abort_flag, 113);
      tc_fence_after();
      const bool whole = seg.j0 == 0 && seg.j1 == seg.n_tiles;
      auto write = [&](int c, const float (&o)[32], float f) {  // dims [c, c + 32)
        if constexpr (kF32) {
          float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + io + c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[i] = make_float4(o[4 * i] * f, o[4 * i + 1] * f, o[4 * i + 2] * f,
                                 o[4 * i + 3] * f);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + io + c);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dst[i] = make_uint4(pack_bf16x2(o[8 * i] * f, o[8 * i + 1] * f),
                                pack_bf16x2(o[8 * i + 2] * f, o[8 * i + 3] * f),
                                pack_bf16x2(o[8 * i + 4] * f, o[8 * i + 5] * f),
                                pack_bf16x2(o[8 * i + 6] * f, o[8 * i + 7] * f));
        }
      };
      float* part = p.part + ((long long)blockIdx.x * 2 + (seg.j0 == 0 ? 1 : 0)) * kTreePartFloats;
      if (warp_real) {
        const float f = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
#pragma unroll 1
        for (int c = 0; c < kD; c += 32) {
          uint32_t w[32];
          tmem_ld32(tmem + lane_off + kColO + c, w);
          tmem_wait_ld();
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(w[i]);
          if (whole) {
            if (real) write(c, o, f);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) part[(c + i) * kRows + r] = o[i];
          }
        }
        if (!whole) {
          part[kD * kRows + r] = m;
          part[kD * kRows + kRows + r] = l;
        }
      }
      tc_fence_before();  // O has been read before the next unit's first P V
      if (!whole) {
        const int c0 = (int)(seg.unit0 / walk.per);
        const int c1 = (int)((seg.unit0 + seg.n_tiles - 1) / walk.per);
        __threadfence();
        named_barrier_sync(1, 128);
        if (tid == 0) {
          const int last = atomicAdd(p.tickets + c0, 1) == c1 - c0;
          if (last) atomicExch(p.tickets + c0, 0);  // re-armed for the next launch
          sm.last = last;
        }
        named_barrier_sync(1, 128);
        const bool last = sm.last;
        named_barrier_sync(1, 128);
        if (last && warp_real) {
          __threadfence();
          auto at = [&](int i) { return p.part + ((long long)i * 2 + (i == c0)) * kTreePartFloats; };
          float M = -INFINITY, L = 0.0f;
          for (int i = c0; i <= c1; ++i) M = fmaxf(M, __ldcg(at(i) + kD * kRows + r));
          for (int i = c0; i <= c1; ++i) {
            const float mi = __ldcg(at(i) + kD * kRows + r);
            const float f = mi == -INFINITY ? 1.0f : fast_exp2(mi - M);
            L = fmaf(__ldcg(at(i) + kD * kRows + kRows + r), f, L);
          }
          const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll 1
          for (int c = 0; c < kD; c += 32) {
            float o[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
            for (int k = c0; k <= c1; ++k) {
              const float* src = at(k);
              const float mk = __ldcg(src + kD * kRows + r);
              const float f = mk == -INFINITY ? 1.0f : fast_exp2(mk - M);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = fmaf(__ldcg(src + (c + i) * kRows + r), f, o[i]);
            }
            if (real) write(c, o, inv);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <bool kF32>
nvattn_status launch(const CUtensorMap& tk, const CUtensorMap& tv, const TreeParams& p, int grid,
                     cudaStream_t stream) {
  const size_t smem = sizeof(TreeSmem) + 1024;
  // (atomic: handles on different threads may launch at the same time)
  static std::atomic<unsigned long long> attr_set_mask{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return NVATTN_ERR_CUDA;
  if (dev >= 64 || !(attr_set_mask.load(std::memory_order_relaxed) & (1ull << dev))) {
    if (cudaFuncSetAttribute(tree_decode_kernel<kF32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem) != cudaSuccess)
      return NVATTN_ERR_CUDA;
    if (dev < 64) attr_set_mask.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  tree_decode_kernel<kF32><<<grid, kThreads, smem, stream>>>(tk, tv, p);
  return cudaGetLastError() == cudaSuccess ? NVATTN_OK : NVATTN_ERR_CUDA;
}

}  // namespace

nvattn_status launch_paged_tree_decode(nvattn_handle* h, int layer, int n_seqs, int n_nodes,
                                       const void* q, nvattn_dtype dtype, const int32_t* cu_nodes,
                                       const uint64_t* mask, int mask_words, int max_nodes,
                                       const uint16_t* k_cache, const uint16_t* v_cache,
                                       const int32_t* block_tables, int max_blocks,
                                       const int32_t* context_lens, int max_context_len,
                                       void* out, cudaStream_t stream) {
  if (n_seqs == 0 || n_nodes == 0) return NVATTN_OK;
  CUtensorMap tk, tv;
  nvattn_status st =
      get_cache_tensor_map(h, k_cache, 64, kTile, CU_TENSOR_MAP_SWIZZLE_128B, &tk);
  if (st != NVATTN_OK) return st;
  st = get_cache_tensor_map(h, v_cache, 64, kTile, CU_TENSOR_MAP_SWIZZLE_128B, &tv);
  if (st != NVATTN_OK) return st;
  TreeParams p = {};
  p.Hq = h->cfg.n_q_heads;
  p.Hkv = h->cfg.n_kv_heads;
  p.G = p.Hq / p.Hkv;
  p.layer = layer;
  p.block_size = h->cfg.block_size;
  p.max_blocks = max_blocks;
  p.n_seqs = n_seqs;
  p.n_nodes = n_nodes;
  p.max_nodes = max_nodes;
  p.mask_words = mask_words;
  p.max_context = max_context_len;
  p.n_slots = h->n_slots;
  p.num_blocks = h->cfg.num_blocks;
  p.scale_log2 = h->cfg.scale * kLog2e;
  p.q = q;
  p.cu_nodes = cu_nodes;
  p.mask = mask;
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.out = out;
  p.part = h->ws_part;
  p.tickets = h->part_tickets;
  p.status = h->status_dev;
  return dtype == NVATTN_DTYPE_BF16 ? launch<false>(tk, tv, p, h->sm_count, stream)
                                    : launch<true>(tk, tv, p, h->sm_count, stream);
}

}  // namespace nvattn
