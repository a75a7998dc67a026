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
// keys then come from L2).  The units' key tiles (kTile keys) are split evenly
// over one CTA per SM (tile_split.cuh); the partials that this makes are
// published at the CTA's end, and the CTA that publishes a unit's last one
// merges them, in CTA order.
//
//   warp 0      TMA producer: K and V tiles (one copy each, the dim halves one
//               after the other, 128-byte swizzle) through two rings of
//               slots that run on across units, and before a unit's first K tile
//               its bf16 queries (box: 64 dims x G heads x 128 / G nodes, the
//               operand's layout) into one of two buffers.
//   warp 1      TMEM allocation; issues S(j) = Q K^T (M = 128 rows, N = kTile
//               keys), up to kBufs tiles ahead, into the next unit too, so that
//               a unit's first scores are there when its softmax starts.
//   warp 2      issues O_w += P V (N = 128 dims, K = kTile keys, A = P from
//               TMEM).  Two issuers, as one spent more time on the waits and
//               commits between the MMAs than on the MMAs.
//   warps 4-11  two groups of four, thread = row = TMEM lane: group w takes
//               the tiles j with j % 2 = w (counted over the run), with its own
//               S / P buffer, running maximum, sum and O_w, so the groups never
//               wait for one another inside a unit, and the tensor cores work
//               on one group's tile while the other group's softmax runs.
//               Online softmax in the log2 domain with lazy rescaling of O_w;
//               P over the columns of its own S.  At a unit's end each group
//               combines O_0 and O_1 for half of the dims.  f32 queries are
//               split into their terms by these warps (one buffer).
// Precision: products of bf16 operands, f32 sums.  bf16 queries are one
// operand and P is a sum of two bf16 terms (16 bits; one term, 8 bits, would
// add as much error as the rounding of a bf16 output itself).  f32 queries and
// their P are sums of three bf16 terms, 24 bits: f32 in, f32 out.
// TMEM columns: O_0 [0, 128), O_1 [128, 256), then the S / P buffers, tile j in
// buffer j % kBufs: P's terms, 32 columns each, over the tile's 64 columns of
// scores.  With four buffers (bf16) a group finds its next scores there while
// its last P V still runs; with two, score, softmax and P V of a group's tiles
// follow one another.
#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "tile_split.cuh"

namespace nvattn {
namespace {

constexpr int kD = 128;
constexpr int kRows = 128;
constexpr int kTile = 64;  // keys per tile (a mask word's)
constexpr int kGroup = 128;  // softmax threads of one group
constexpr int kThreads = 3 * kGroup;
// Registers per thread: 168 at launch (384 threads); the softmax groups take
// what warps 0-3 give up: 88 + 2 * 208 = 3 * 168.
constexpr int kControlRegs = 88, kSoftmaxRegs = 208;
constexpr int kQTermBytes = kRows * kD * 2;     // [d half][row][64], 128-byte swizzle
constexpr int kOperandBytes = 13 * 16 * 1024;  // query operands and the ring share it
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 256;  // the S / P buffers; O_0 and O_1 lie before them
constexpr float kLog2e = 1.4426950408889634f;
// log2: a row's reference moves only when a score passes it by 2^32.  P, O and
// the sums are floating point, so weights above 1 lose nothing, and f32 leaves
// 2^90 for the values.
constexpr float kSlack = 32.0f;
// A unit's end costs about as much as this many keys, and the split counts
// them.
constexpr int kUnitCostKeys = 512;
// Fewest keys per CTA: below that a CTA's own start and the merge of more
// partials cost more than the tiles.
constexpr int kMinRunKeys = 128;

struct TreeParams {
  int Hq, Hkv, G, layer, block_size, max_blocks, n_seqs, n_nodes, max_nodes, mask_words;
  int max_context, row_tiles;  // row_tiles: of a sequence of max_nodes
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

// A sequence's nodes and context; n = 0 where it has none or its metadata is
// unusable (`report`: recorded then).
struct SeqInfo {
  int node0, n, ctx;
};
// The units' order: row tile by row tile, each over all sequences and their kv
// heads (entry e of the line: row tile e / n_seqs of sequence e % n_seqs).  The
// row tiles of a kv head then lie a large part of the line apart, where other
// CTAs read the same keys at about the same time, mostly from L2; one after
// another they would be read by one CTA, the second time from memory.
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
__device__ __forceinline__ SeqInfo entry_info(const TreeParams& p, int e) {
  SeqInfo i = seq_info(p, e % p.n_seqs, false);
  if ((e / p.n_seqs) * kRows >= i.n * p.G) i.n = 0;  // no such row tile
  return i;
}
__device__ __forceinline__ int key_tiles(int ctx) {
  return (ctx + kTile - 1) / kTile;
}

// One unit's part of the CTA's run: key tiles [j0, j1).
struct Segment {
  int seq, head, row_tile, j0, j1, n_tiles;
  SeqInfo info;
  int unit0;  // place of the unit's first tile
};

constexpr int kMaxSlots = 13;
struct __align__(1024) TreeSmem {
  uint8_t operands[kOperandBytes];  // query terms, then the K slots, then the V slots
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t q_full[2], q_empty[2], s_full[4], p_full[4], o_done;
  float m[2][kRows], l[2][kRows];  // the groups' references and sums at a unit's end
  // [group][tile with nodes, mod 3]: keys whose V row holds a NaN or an infinity
  uint32_t bad[2][3][kTile / 32];
  uint32_t tmem_base;
  int abort_flag;
  int skip;
  int last[2];
  Segment shared[2];  // units shared with other CTAs: at most the run's ends
  int per;            // places per CTA
};
static_assert(sizeof(TreeSmem) + 1024 <= 227 * 1024, "shared memory");

// Walks the segments of a run; every role walks the same ones.
struct Walker {
  static constexpr int kUnitCost = kUnitCostKeys / kTile;
  int at, end;
  int entry, head;  // the unit that `at` lies in
  int offset;       // place of `at` in its unit
  SeqInfo info;

  __device__ __forceinline__ void start(const TreeParams& p, const tilesplit::Run& r) {
    at = r.begin;
    end = r.end;
    entry = r.seq;
    if (at >= end) return;
    info = entry_info(p, entry);
    const int span = key_tiles(info.ctx) + kUnitCost;
    head = (at - r.seq_first) / span;
    offset = (at - r.seq_first) % span;
  }

  __device__ __forceinline__ bool next(const TreeParams& p, Segment& s) {
    while (at < end) {
      const int tiles = key_tiles(info.ctx);
      const int left = tiles + kUnitCost - offset;
      const int take = min(left, end - at);
      const int j0 = max(offset - kUnitCost, 0), j1 = offset + take - kUnitCost;
      const bool some = j1 > j0;
      if (some)
        s = {entry % p.n_seqs, head, entry / p.n_seqs, j0, j1, tiles, info,
             at - offset + kUnitCost};
      at += take;
      offset = 0;
      if (take == left && at < end && ++head == p.Hkv) {
        head = 0;
        do info = entry_info(p, ++entry);
        while (info.n == 0);  // (`at` < end: a later entry has places)
      }
      if (some) return true;
    }
    return false;
  }
};

// kN consecutive dims of an output row at element `at`, times f.
template <bool kF32, int kN>
__device__ __forceinline__ void write_dims(const TreeParams& p, long long at, const float (&o)[kN],
                                           float f) {
  if constexpr (kF32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
#pragma unroll
    for (int i = 0; i < kN / 4; ++i)
      dst[i] = make_float4(o[4 * i] * f, o[4 * i + 1] * f, o[4 * i + 2] * f, o[4 * i + 3] * f);
  } else {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at);
#pragma unroll
    for (int i = 0; i < kN / 8; ++i)
      dst[i] = make_uint4(pack_bf16x2(o[8 * i] * f, o[8 * i + 1] * f),
                          pack_bf16x2(o[8 * i + 2] * f, o[8 * i + 3] * f),
                          pack_bf16x2(o[8 * i + 4] * f, o[8 * i + 5] * f),
                          pack_bf16x2(o[8 * i + 6] * f, o[8 * i + 7] * f));
  }
}

// 32 dims from `d` of 32 rows of a unit's sequence, rows row0 + lane (those
// below n_rows).  Lanes trade 16-byte chunks in fours, so that four of them
// write 64 consecutive bytes of one row: a lane alone would write 16 bytes to
// a line of its own.
template <bool kF32>
__device__ __forceinline__ void write_rows(const TreeParams& p, const Segment& seg, int row0,
                                           int n_rows, int d, const float (&o)[32]) {
  constexpr int kPer = kF32 ? 4 : 8;  // elements per chunk
  const int lane = threadIdx.x & 31, log_g = 31 - __clz(p.G);
#pragma unroll
  for (int set = 0; set < 32; set += 4 * kPer) {
    uint32_t u[4][4];  // [chunk], then [row of the four]
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int x = set + kPer * i + e * (kPer / 4);
        u[i][e] = kF32 ? __float_as_uint(o[x]) : pack_bf16x2(o[x], o[x + kPer / 4 - 1]);
      }
#pragma unroll
    for (int stage = 1; stage <= 2; ++stage) {
      const bool odd = lane & stage;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i & stage) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t &a = u[i][e], &b = u[i | stage][e];
          const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? a : b, stage);
          if (odd) a = other; else b = other;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + (lane & ~3) + i;
      if (row < n_rows) {
        const long long at = ((long long)(seg.info.node0 + (row >> log_g)) * p.Hq +
                              (long long)seg.head * p.G + (row & (p.G - 1))) * kD +
                             d + set + kPer * (lane & 3);
        *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + at * (kF32 ? 4 : 2)) =
            make_uint4(u[i][0], u[i][1], u[i][2], u[i][3]);
      }
    }
  }
}

// A softmax warp's share of `rows` rows of 128 dims: a lane per row, `dims` dims
// from d0.  Where the rows are few the eight warps split the dims.
struct Share {
  int row, d0, dims;
};
__device__ __forceinline__ Share share_of(int rows) {
  const int w = ((int)threadIdx.x >> 5) - 4;  // 0..7
  const int quads = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  const int dims = kD * quads / 8;
  return {(w % quads) * 32 + ((int)threadIdx.x & 31), (w / quads) * dims, dims};
}

// Merges the partials of a unit that CTAs c0..c1 share, in CTA order: split
// over the softmax warps (share_of).
// Four partials at a time, with all of their loads in flight together: the
// reads are bound by their latency where the rows are few, and by what one SM
// reads from L2 (about 110 GB/s) where they are many.
template <bool kF32>
__device__ __forceinline__ void merge_parts(const TreeParams& p, const Segment& seg, int c0,
                                            int c1) {
  constexpr int kAtOnce = 4, kDims = 16;
  const int rows = min(seg.info.n * p.G - seg.row_tile * kRows, kRows);
  const Share share = share_of(rows);
  const int r = share.row;
  if (r >= rows) return;
  const int row = seg.row_tile * kRows + r;
  const long long io = ((long long)(seg.info.node0 + row / p.G) * p.Hq +
                        (long long)seg.head * p.G + row % p.G) * kD;
#pragma unroll 1
  for (int d = share.d0; d < share.d0 + share.dims; d += kDims) {
    float o[kDims], M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int i = 0; i < kDims; ++i) o[i] = 0.0f;
#pragma unroll 1
    for (int k = c0; k <= c1; k += kAtOnce) {
      float v[kAtOnce][kDims], m[kAtOnce], l[kAtOnce];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        m[e] = -INFINITY;
        if (k + e > c1) continue;
        // (the first CTA left its part in its second place: tile_split.cuh)
        const int i = k + e;
        const float* src = p.part + ((long long)i * 2 + (i == c0)) * kTreePartFloats + r;
        m[e] = __ldcg(src + kD * kRows);
        l[e] = __ldcg(src + kD * kRows + kRows);
#pragma unroll
        for (int j = 0; j < kDims; ++j) v[e][j] = __ldcg(src + (d + j) * kRows);
      }
      const float top = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), M);
      const float old = M == -INFINITY ? 1.0f : fast_exp2(M - top);
      M = top;
      L *= old;
#pragma unroll
      for (int j = 0; j < kDims; ++j) o[j] *= old;
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        if (k + e > c1) break;
        const float f = m[e] == -INFINITY ? 1.0f : fast_exp2(m[e] - top);
        L = fmaf(l[e], f, L);
#pragma unroll
        for (int j = 0; j < kDims; ++j) o[j] = fmaf(v[e][j], f, o[j]);
      }
    }
    write_dims<kF32, kDims>(p, io + d, o, L == 0.0f ? 0.0f : 1.0f / L);
  }
}

// kF32: f32 queries and outputs (three terms each), else bf16 (one and two).
template <bool kF32>
__global__ void __launch_bounds__(kThreads, 1)
    tree_decode_kernel(const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ CUtensorMap tm_q, TreeParams p) {
  constexpr int kT = kTile, kTileBytes = kT * kD * 2;
  constexpr int kHalfBytes = kTileBytes / 2;  // one box: kT tokens x 64 dims
  constexpr int kQ = kF32 ? 3 : 1, kP = kF32 ? 3 : 2;
  constexpr int kQBufs = kF32 ? 1 : 2;
  constexpr int kQBytes = kQBufs * kQ * kQTermBytes;
  // S / P buffers: four for bf16, two where P has three terms
  constexpr int kBufs = kF32 ? 2 : 4;
  constexpr int kSlotsK = kF32 ? 3 : 4, kSlotsV = kF32 ? 4 : 5;
  static_assert(kQBytes + (kSlotsK + kSlotsV) * kTileBytes <= kOperandBytes &&
                kSlotsK + kSlotsV <= kMaxSlots, "ring");
  // P V(t) is waited for on V(t)'s `empty` barrier, by the S issuer at tile t +
  // kBufs and by the softmax at t + 2.  The slot's next use ends with P V(t +
  // kSlotsV), which comes after that waiter's own tile's (P Vs are issued in
  // order), so the barrier cannot be two uses ahead of the wait.
  static_assert(kSlotsV >= kBufs && kSlotsV >= 2, "V slots");
  constexpr uint32_t kColsS = 256 / kBufs;
  static_assert(kT <= (int)kColsS && kP * kT / 2 <= (int)kColsS, "TMEM columns");
  extern __shared__ uint8_t smem_raw[];
  TreeSmem& sm = *reinterpret_cast<TreeSmem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = sm.operands + kQBytes;
  // slots of tile g's K and V, and the parity of their use
  auto k_slot = [](int g) { return g % kSlotsK; };
  auto k_parity = [](int g) { return (uint32_t)(g / kSlotsK) & 1u; };
  auto v_slot = [](int g) { return kSlotsK + g % kSlotsV; };
  auto v_parity = [](int g) { return (uint32_t)(g / kSlotsV) & 1u; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    if constexpr (!kF32) tma_prefetch_desc(&tm_q);
    for (int i = 0; i < kSlotsK + kSlotsV; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], kF32 ? 8 : 1);
      mbar_init(&sm.q_empty[i], 1);
      for (int k = 0; k < 3; ++k) sm.bad[i][k][0] = sm.bad[i][k][1] = 0;
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
    }
    mbar_init(&sm.o_done, 1);
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
  Walker walk;
  const tilesplit::Run run =
      tilesplit::find_run(p.n_seqs * p.row_tiles, blockIdx.x, gridDim.x, kMinRunKeys / kT,
                          [&](int e) {
                            const SeqInfo i = entry_info(p, e);
                            return tilesplit::SeqTiles{i.n > 0 ? p.Hkv : 0,
                                                       key_tiles(i.ctx) + Walker::kUnitCost};
                          });
  walk.start(p, run);
  if (threadIdx.x == 0) sm.per = run.per;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_flag = &sm.abort_flag;
  if (sm.skip) walk.at = walk.end;
  Segment seg;

  if (warp < 4) {
    regs_dec<kControlRegs>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- producer
      // (evict_first also where a kv head has several row tiles, whose reads
      // come close together: 16 ragged drafts took 109 us with it, 117 without)
      const uint64_t policy = l2_policy_evict_first();
      int g = 0;
      for (int n_seg = 0; walk.next(p, seg); ++n_seg) {
        if constexpr (!kF32) {
          const int b = n_seg & 1;
          if (n_seg >= 2)
            mbar_wait(&sm.q_empty[b], ((n_seg >> 1) - 1) & 1, p.status, abort_flag, 114);
          uint8_t* dst = sm.operands + b * kQTermBytes;
          const int node = seg.info.node0 + seg.row_tile * (kRows / p.G);
          mbar_arrive_expect_tx(&sm.q_full[b], kQTermBytes);
          tma_load_3d(dst, &tm_q, &sm.q_full[b], 0, seg.head * p.G, node);
          tma_load_3d(dst + kQTermBytes / 2, &tm_q, &sm.q_full[b], 64, seg.head * p.G, node);
        }
        int block = -1;
        long long bid = 0;
        for (int j = seg.j0; j < seg.j1; ++j, ++g) {
          const int tok = j * kT;
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
            const int slot = kv ? v_slot(g) : k_slot(g);
            if (g >= (kv ? kSlotsV : kSlotsK))
              mbar_wait(&sm.empty[slot], (kv ? v_parity(g) : k_parity(g)) ^ 1u, p.status,
                        abort_flag, 103);
            mbar_arrive_expect_tx(&sm.full[slot], kTileBytes);
            tma_load_4d_hint(ring + slot * kTileBytes, kv ? &tm_v : &tm_k, &sm.full[slot], 0,
                             seg.head, row, 0, policy);
          }
        }
      }
      // Drain: the last load of every slot has landed before the CTA exits
      // (the query loads precede them, and the MMAs have waited for those).
      for (int i = max(0, g - kSlotsK); i < g; ++i)
        mbar_wait(&sm.full[k_slot(i)], k_parity(i), p.status, 104);
      for (int i = max(0, g - kSlotsV); i < g; ++i)
        mbar_wait(&sm.full[v_slot(i)], v_parity(i), p.status, 104);
    }
    // ------------------------------------------------------------ MMA issuers
    // (each warp runs converged, so that descriptors and loop values stay
    // warp-uniform, and elects a lane at each tcgen05 instruction: issued from
    // a one-lane branch an MMA took ~125 cycles, so ~50)
    auto commit = [](uint64_t* bar) {
      if (elect_one()) umma_commit(bar);
    };
    if (warp == 1) {
      constexpr uint32_t idesc = umma_idesc_bf16_f32(kRows, kT, 0, 0);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(sm.operands), 16, 1024);
      const uint64_t k_desc = umma_desc_sw128(smem_u32(ring), 16, 1024);
      int g = 0;
      for (int n_seg = 0; walk.next(p, seg); ++n_seg) {
        const int n = seg.j1 - seg.j0, qb = n_seg % kQBufs;
        mbar_wait(&sm.q_full[qb], (n_seg / kQBufs) & 1, p.status, abort_flag, 105);
        const uint64_t qd = q_desc + (uint64_t)(qb * (kQTermBytes / 16));
        for (int j = 0; j < n; ++j, ++g) {
          const int slot = k_slot(g), prev = g - kBufs;
          mbar_wait(&sm.full[slot], k_parity(g), p.status, abort_flag, 106);
          if (prev >= 0)  // P V of the buffer's last tile is complete
            mbar_wait(&sm.empty[v_slot(prev)], v_parity(prev), p.status, abort_flag, 115);
          tc_fence_after();
          const uint64_t kd = k_desc + (uint64_t)(slot * (kTileBytes / 16));
          const uint32_t d = tmem + kColS + (g % kBufs) * kColsS;
#pragma unroll
          for (int t = kQ - 1; t >= 0; --t)  // the small terms first
#pragma unroll
            for (int k = 0; k < kD / 16; ++k)
              if (elect_one())
                umma_bf16(d,
                          qd + (uint64_t)((t * kQTermBytes + (k >> 2) * (kQTermBytes / 2) +
                                           (k & 3) * 32) / 16),
                          kd + (uint64_t)(((k >> 2) * kHalfBytes + (k & 3) * 32) / 16), idesc,
                          (t < kQ - 1 || k > 0) ? 1u : 0u);
          commit(&sm.s_full[g % kBufs]);
          commit(&sm.empty[slot]);
        }
        commit(&sm.q_empty[qb]);
      }
    } else if (warp == 2) {
      constexpr uint32_t idesc = umma_idesc_bf16_f32(kRows, kD, 0, 1);
      const uint64_t v_desc = umma_desc_sw128(smem_u32(ring), kHalfBytes, 1024);
      int g = 0, n_seg = 0;
      for (; walk.next(p, seg); ++n_seg) {
        const int n = seg.j1 - seg.j0;
        for (int j = 0; j < n; ++j, ++g) {
          const int slot = v_slot(g);
          mbar_wait(&sm.p_full[g % kBufs], (g / kBufs) & 1, p.status, abort_flag, 107);
          mbar_wait(&sm.full[slot], v_parity(g), p.status, abort_flag, 108);
          tc_fence_after();
          const uint32_t a = tmem + kColS + (g % kBufs) * kColsS;
          const uint64_t vd = v_desc + (uint64_t)(slot * (kTileBytes / 16));
#pragma unroll
          for (int t = kP - 1; t >= 0; --t)
#pragma unroll
            for (int k = 0; k < kT / 16; ++k)
              if (elect_one())
                umma_bf16_ts(tmem + (g & 1) * kD,
                             a + 32 * t + 8 * k,
                             vd + (uint64_t)(k * 16 * 128 / 16), idesc,
                             (j > 1 || t < kP - 1 || k > 0) ? 1u : 0u);
          commit(&sm.empty[slot]);
        }
        commit(&sm.o_done);
      }
      // Drain: every MMA has completed before TMEM is released (each S has
      // been waited for by the softmax before its P V).
      if (n_seg > 0) mbar_wait(&sm.o_done, (n_seg - 1) & 1, p.status, 109);
    }
  } else {
    // ------------------------------------------------------------ softmax
    regs_inc<kSoftmaxRegs>();
    const int grp = (warp - 4) >> 2;  // group
    const int tid = (int)threadIdx.x & (kGroup - 1);
    const int quad = warp & 3;  // TMEM lanes [32 * quad, 32 * quad + 32)
    const int r = quad * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t o_col = lanes + grp * kD;
    const uint64_t c2 = pack2(p.scale_log2, p.scale_log2);
    int g = 0;  // tiles of the run before the segment
    int n_shared = 0;
    int n_special = 0;  // tiles with nodes (of this group) so far
    bool more = walk.next(p, seg);
    for (int n_seg = 0; more; ++n_seg) {
      const int n_rows = seg.info.n * p.G;
      const int row = seg.row_tile * kRows + r;
      const bool real = row < n_rows;
      const bool warp_real = seg.row_tile * kRows + quad * 32 < n_rows;
      const int node = seg.info.node0 + (real ? row / p.G : 0);
      const int first = seg.info.ctx - seg.info.n;  // position of the sequence's first node
      if constexpr (kF32) {
        // ---- query operand (the MMAs that read the last one are complete:
        // o_done), 16 dims at a time ----
        const int q_rows = min(n_rows - seg.row_tile * kRows, kRows);
        const Share share = share_of(q_rows);
        if ((share.row & ~31) < q_rows) {
          const bool q_real = share.row < q_rows;
          const int q_row = seg.row_tile * kRows + (q_real ? share.row : 0);
          const float4* src = reinterpret_cast<const float4*>(
              static_cast<const float*>(p.q) +
              ((long long)(seg.info.node0 + q_row / p.G) * p.Hq + (long long)seg.head * p.G +
               q_row % p.G) * kD + share.d0);
          uint8_t* dst = sm.operands + share.row * 128;
          float4 next[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) next[i] = src[i];
#pragma unroll 1
          for (int d = 0; d < share.dims; d += 16) {
            float4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = q_real ? next[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              if (d + 16 < share.dims) next[i] = src[(d + 16) / 4 + i];
            }
            uint8_t* half = dst + ((share.d0 + d) >> 6) * (kQTermBytes / 2);
            const int chunk = ((share.d0 + d) & 63) >> 3;  // of 8 dims
#pragma unroll
            for (int t = 0; t < kQ; ++t)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint4 w;
                split_term(v[2 * i].x, v[2 * i].y, w.x);
                split_term(v[2 * i].z, v[2 * i].w, w.y);
                split_term(v[2 * i + 1].x, v[2 * i + 1].y, w.z);
                split_term(v[2 * i + 1].z, v[2 * i + 1].w, w.w);
                *reinterpret_cast<uint4*>(half + t * kQTermBytes +
                                          (((chunk + i) ^ (share.row & 7)) << 4)) = w;
              }
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[0]);
      }

      float m = -INFINITY, l = 0.0f;
      const int n = seg.j1 - seg.j0;
      const int j_first = (grp ^ g) & 1;  // the group's first tile of the segment
      for (int j = j_first; j < n; j += 2) {
        const int gj = g + j;
        const int col0 = (seg.j0 + j) * kT;
        const uint32_t s_col = lanes + kColS + (gj % kBufs) * kColsS;
        const bool special = col0 + kT > first;  // the tile holds nodes (or keys past the end)
        uint64_t allowed = 0;                    // which of its keys the row attends
        if (special) {  // (before the wait for its scores, which it hides behind)
          const int rel = col0 - first;  // the first key's place among the nodes, > -kT
          if (real) {
            const uint64_t* words = p.mask + (long long)node * p.mask_words;
            if (rel < 0) {
              allowed = (words[0] << -rel) | ((1ull << -rel) - 1);
            } else {
              const int q = rel >> 6, sh = rel & 63;
              if (q < p.mask_words) allowed = words[q] >> sh;
              if (sh > 0 && q + 1 < p.mask_words) allowed |= words[q + 1] << (64 - sh);
            }
          }
          const int here = seg.info.ctx - col0;  // keys of the context from here on
          if (here < kT) allowed &= (1ull << here) - 1;
          // V rows of nodes that hold a NaN or an infinity: 0 * NaN would
          // reach the rows whose masks leave the node out.  Such a row is
          // zeroed and noted, and makes the rows that attend it NaN.  Slots
          // past the context may hold anything and are zeroed.
          const int slot = v_slot(gj);
          mbar_wait(&sm.full[slot], v_parity(gj), p.status, abort_flag, 111);
          volatile uint32_t* bad_now = sm.bad[grp][n_special % 3];
          {
            const int t = tid >> 1;  // key of the tile; two threads, a dim half each
            uint4* v = reinterpret_cast<uint4*>(ring + slot * kTileBytes + (tid & 1) * kHalfBytes +
                                                t * 128);
            const bool past = col0 + t >= seg.info.ctx;
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint4 c = v[k];
              const uint32_t u[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                bad = bad || (u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u;
            }
            const uint32_t votes = __ballot_sync(0xffffffffu, bad && !past && col0 + t >= first);
            bad = (votes >> (lane & ~1)) & 3u;
            if (bad && (tid & 1) == 0)
              atomicOr(&sm.bad[grp][n_special % 3][t >> 5], 1u << (t & 31));
            if (bad || past) {
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();
          named_barrier_sync(1 + grp, kGroup);
          const uint64_t bad_keys = (uint64_t)bad_now[1] << 32 | bad_now[0];
          if (bad_keys & allowed) l = __uint_as_float(0x7fc00000u);
          // Cleared for the tile with nodes after the next one: every thread has
          // read it (before this barrier), and none sets it before the next one.
          if (tid < 2) sm.bad[grp][(n_special + 2) % 3][tid] = 0;
          ++n_special;
        }
        mbar_wait(&sm.s_full[gj % kBufs], (gj / kBufs) & 1, p.status, abort_flag, 110);
        tc_fence_after();
        if (warp_real) {
          float x[kT];
#pragma unroll
          for (int c = 0; c < kT; c += 32)
            tmem_ld32(s_col + c, *reinterpret_cast<uint32_t(*)[32]>(&x[c]));
          tmem_wait_ld();
          if (special) {
#pragma unroll
            for (int i = 0; i < kT; ++i)
              x[i] = (allowed >> i) & 1 ? x[i] : -INFINITY;
          }
          float tops[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int i = 4; i + 4 < kT; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) tops[e] = fmax3(tops[e], x[i + e], x[i + 4 + e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) tops[e] = fmaxf(tops[e], x[kT - 4 + e]);
          const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * p.scale_log2;
          if (__any_sync(0xffffffffu, top > m + kSlack)) {
            // (the first tile of a unit, hardly ever again)  A new reference;
            // the sums and O_w so far are rescaled.
            const float m_new = top > m + kSlack ? top : m;
            const float alpha = m_new == m ? 1.0f : fast_exp2(m - m_new);  // m = -inf: 0
            m = m_new;
            l *= alpha;
            if (j > j_first) {
              // P V(j - 2), the group's last, must be complete: its V is free
              mbar_wait(&sm.empty[v_slot(gj - 2)], v_parity(gj - 2), p.status, abort_flag, 112);
              tc_fence_after();
#pragma unroll 1
              for (int d = 0; d < kD; d += 16) {
                uint32_t w[16];
                tmem_ld16(o_col + d, w);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  w[i] = __float_as_uint(__uint_as_float(w[i]) * alpha);
                tmem_st16(o_col + d, w);
              }
              tmem_wait_st();
            }
          }
          const float ref = m == -INFINITY ? 0.0f : m;  // a row without keys yet: weights 0
          const uint64_t r2 = pack2(-ref, -ref);
          uint64_t s2[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < kT / 2; ++i) {
            float a, b;
            unpack2(ffma2(pack2(x[2 * i], x[2 * i + 1]), c2, r2), a, b);
            x[2 * i] = fast_exp2(a);
            x[2 * i + 1] = fast_exp2(b);
            s2[i & 1] = fadd2(s2[i & 1], pack2(x[2 * i], x[2 * i + 1]));
          }
#pragma unroll
          for (int t = 0; t < kP; ++t) {
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) split_term(x[2 * i], x[2 * i + 1], w[i]);
            tmem_st32(s_col + 32 * t, w);
          }
          float s0, s1, s3, s4;
          unpack2(s2[0], s0, s1);
          unpack2(s2[1], s3, s4);
          l += (s0 + s1) + (s3 + s4);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[gj % kBufs]);
      }
      g += n;

      // ---- the unit's end: each group combines O_0 and O_1 for half of the dims ----
      sm.m[grp][r] = m;
      sm.l[grp][r] = l;
      Segment next_seg;
      more = walk.next(p, next_seg);  // (while the last P V runs)
      mbar_wait(&sm.o_done, n_seg & 1, p.status, abort_flag, 113);
      tc_fence_after();
      named_barrier_sync(3, 2 * kGroup);
      const bool whole = seg.j0 == 0 && seg.j1 == seg.n_tiles;
      float* part = p.part + ((long long)blockIdx.x * 2 + (seg.j0 == 0 ? 1 : 0)) * kTreePartFloats;
      if (warp_real) {
        const float m0 = sm.m[0][r], m1 = sm.m[1][r];
        const float M = fmaxf(m0, m1);
        const float f0 = m0 == -INFINITY ? 1.0f : fast_exp2(m0 - M);
        const float f1 = m1 == -INFINITY ? 1.0f : fast_exp2(m1 - M);
        const float L = fmaf(sm.l[1][r], f1, sm.l[0][r] * f0);
        const float inv = whole ? (L == 0.0f ? 0.0f : 1.0f / L) : 1.0f;  // no key: zeros
        // a segment of one tile has written only one of the two
        const bool has0 = n > 1 || ((g - 1) & 1) == 0, has1 = n > 1 || ((g - 1) & 1) == 1;
#pragma unroll 1
        for (int c = 64 * grp; c < 64 * grp + 64; c += 32) {
          float o[32];
          uint32_t w0[32], w1[32];
          if (has0) tmem_ld32(lanes + c, w0);
          if (has1) tmem_ld32(lanes + kD + c, w1);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            o[i] = ((has0 ? __uint_as_float(w0[i]) * f0 : 0.0f) +
                    (has1 ? __uint_as_float(w1[i]) * f1 : 0.0f)) * inv;
          if (whole) {
            write_rows<kF32>(p, seg, seg.row_tile * kRows + quad * 32, n_rows, c, o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) part[(c + i) * kRows + r] = o[i];
          }
        }
        if (!whole && grp == 0) {
          part[kD * kRows + r] = M;
          part[kD * kRows + kRows + r] = L;
        }
      }
      // Neither group goes on before the other has read both O, both sums and
      // o_done: its next P would start the next unit's P V over them.
      tc_fence_before();
      named_barrier_sync(3, 2 * kGroup);
      if (!whole) {
        if (threadIdx.x == kGroup) sm.shared[n_shared] = seg;
        ++n_shared;
      }
      seg = next_seg;
    }
    // ---- publish the partials; merge the units whose last one this is ----
    if (n_shared > 0) {
      __threadfence();
      named_barrier_sync(3, 2 * kGroup);
      auto ctas = [&](const Segment& u, int& c0, int& c1) {
        c0 = u.unit0 / sm.per;
        c1 = (u.unit0 + u.n_tiles - 1) / sm.per;
      };
      int c0, c1;
      if (tid < n_shared && grp == 0) {
        ctas(sm.shared[tid], c0, c1);
        const int last = atomicAdd(p.tickets + c0, 1) == c1 - c0;
        if (last) atomicExch(p.tickets + c0, 0);  // re-armed for the next launch
        sm.last[tid] = last;
      }
      named_barrier_sync(3, 2 * kGroup);
#pragma unroll 1
      for (int i = 0; i < n_shared; ++i)
        if (sm.last[i]) {
          __threadfence();
          ctas(sm.shared[i], c0, c1);
          merge_parts<kF32>(p, sm.shared[i], c0, c1);
        }
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <bool kF32>
nvattn_status launch(const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq,
                     const TreeParams& p, int grid, cudaStream_t stream) {
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
  tree_decode_kernel<kF32><<<grid, kThreads, smem, stream>>>(tk, tv, tq, p);
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
  const bool bf16 = dtype == NVATTN_DTYPE_BF16;
  CUtensorMap tk, tv, tq = {};
  nvattn_status st = get_cache_tile_map(h, k_cache, kTile, &tk);
  if (st != NVATTN_OK) return st;
  st = get_cache_tile_map(h, v_cache, kTile, &tv);
  if (st != NVATTN_OK) return st;
  if (bf16) {
    // a unit's 128 query rows: G heads of 128 / G nodes (rows past the batch
    // read as zeros; those of a later sequence are computed and not written)
    const uint64_t Hq = (uint64_t)h->cfg.n_q_heads;
    const int G = h->cfg.n_q_heads / h->cfg.n_kv_heads;
    st = encode_tensor_map_3d(&tq, q, kD, Hq, (uint64_t)n_nodes, kD * 2, Hq * kD * 2, 64,
                              (uint32_t)G, (uint32_t)(kRows / G), CU_TENSOR_MAP_SWIZZLE_128B);
    if (st != NVATTN_OK) return st;
  }
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
  p.row_tiles = (max_nodes * p.G + kRows - 1) / kRows;
  if ((long long)n_seqs * p.row_tiles * p.Hkv *
          ((long long)max_context_len / kTile + 1 + Walker::kUnitCost) >= tilesplit::kMaxPlaces)
    return NVATTN_ERR_UNSUPPORTED;
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
  return bf16 ? launch<false>(tk, tv, tq, p, h->sm_count, stream)
              : launch<true>(tk, tv, tq, p, h->sm_count, stream);
}

}  // namespace nvattn
