// decode_q8.cu -- paged GQA decode attention over the 8-bit KV cache.
//
//   o = sum_t softmax_t(scale * s_k[t] * q.K8[t]) * s_v[t] * V8[t]
//
// K8, V8: e4m3 rows of 128, s_k, s_v: their power-of-two scales; pages
// [layer][block][kv head][token][128], so a (block, kv head) is one contiguous
// run of both.  Both scales leave the matrix products: s_k multiplies the
// score, and s_v joins the exponent,
//   x_t = scale * log2(e) * s_k[t] * (q.K8[t]) + log2 s_v[t]
//   w_t = 2^(x_t - M),  o = sum w_t V8[t] / sum w_t / s_v[t],  M >= x_t - 8
// A key with a large weight may add nothing to the output, or nothing to most
// of its dims (a V row of zeros, which has scale 1; an attention sink with a
// small V row; a row with one large dim), while it is the others, far below it,
// that make the output.  So a weight keeps all of its bits however small it is
// next to the largest: it goes to the tensor cores as a sum of three bf16
// terms, 24 bits and f32's range.  (As an f16 value and its f16 remainder, two
// products instead of three, it had an absolute floor of 2^-25: a zero row
// beside rows of size 0.01 cost the output 8e-4 of its value, a zero row 12 nats
// above 9,000 others 0.3.  The third product costs 10 of the 156 us of 64 long
// f32 sequences, the bf16 operands 7.)
//
// Bound by memory (264 bytes per cached token and kv head against 2 * 128 * 2
// products per query head), and near it by the chain of a step's products and
// exponentials.  The rows of one kv head are at most eight, so the products run
// transposed as mma.sync m16n8k16: tokens or dims in M, the query rows in N = 8.
// A 128-row tcgen05 tile could not use its rows, and the 8-bit rows go from
// shared memory through registers without the widened copy in shared memory
// that a tcgen05 operand would need.
//   K: f16, which holds e4m3 exactly, one conversion for two values.  The
//      queries are scaled to f16's upper range: bf16 ones are f16 values then,
//      f32 ones a value and its remainder times 2^11, whose products are summed
//      apart (22 bits of a query down to 2^-28 of its row's largest).
//   V: bf16, where an e4m3 byte's exponent and mantissa, moved to bf16's place,
//      are its value times 2^-120 (subnormals included): a byte permutation that
//      extends the sign, a shift and a mask.  The weights make up for 2^100 of
//      that, so that products and sums stay normal, the output for the rest.
//
// Each warp works alone: 32-token steps, K and V tiles of 4 KiB each by TMA
// (128-byte swizzle) and their scales by bulk copies into its own ring of
// kStages, its own running reference M, sum and output.  A CTA's kWarps warps
// take consecutive 32-token steps of a 128-token tile; the CTAs' tiles are
// split evenly (tile_split.cuh).  At a unit's end the warps' results are
// merged in shared memory, and where CTAs share a unit the last of them to
// finish merges their partials in CTA order (the same sums on every run).
//
// Which lane reads what.  Token n of a group of eight is row (n >> 1) |
// (n & 1) << 2 of the group, and of the 16-byte chunks of a V row lane group g
// takes chunk (g >> 1) | (g & 1) << 2: with the swizzle that makes every
// 16-byte shared load of a quarter warp hit 32 distinct banks.  A lane's 16
// bytes of K feed four products (the dimension order inside a dot product is
// free, and the query operand uses the same order); of V, eight products of
// two dimensions each, after pairing the bytes of two tokens.  The weights
// turn from the scores' layout into an operand by movmatrix.
#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "tile_split.cuh"

namespace nvattn {
namespace {

constexpr int kD = 128;
constexpr int kWarps = kQ8Warps;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 32;                // tokens per warp step
constexpr int kTile = kWarps * kStep;    // tokens per CTA tile
constexpr int kStages = 2;
constexpr int kRows = 8;                 // query rows per unit (GQA group, padded)
static_assert(kRows == 2 * kWarps, "merge_parts: two rows per warp");
// A unit's start and end (its queries, the warps' merge, its rows or partial)
// cost about as much as this many tiles, and the split counts them as such.
constexpr int kUnitCost = 2;
// Three CTAs per SM hide more of a warp's own latencies (64 sequences of 1k to
// 16k tokens, f32: 156 us, two: 164), two make fewer partials and merges (24 ragged
// batches of 10 to 35 us: 5 to 8 % less in the mean).  Three where the batch may
// hold so many tiles per CTA, by the host's bound of the contexts.
constexpr int kFullGridTiles = 48;
// Shared memory of a launch with two CTAs per SM: more than a third of an SM's,
// so that no SM takes three while another takes one.
constexpr size_t kTwoCtaSmem = 96 * 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;           // log2: rescale only past 2^8
static_assert(128 % kStep == 0, "a step must not cross a block (block sizes are multiples of 128)");

struct Q8Params {
  int Hq, Hkv, G, layer, block_size, max_blocks, n_seqs, max_context;
  long long num_blocks;
  float scale_log2;
  const void* q;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* context_lens;
  void* out;
  float* part;   // [CTA][2][kQ8PartFloats]
  int* tickets;  // [CTA], zero between launches
  DeviceStatus* status;
};

struct __align__(1024) WarpRing {
  uint8_t k[kStages][kStep * kD];
  uint8_t v[kStages][kStep * kD];
};

struct __align__(1024) Q8Smem {
  WarpRing ring[kWarps];
  float ks[kWarps][kStages][kStep];
  float vs[kWarps][kStages][kStep];
  float4 tok[kWarps][kStep];  // {score factor, log2 s_v, 1 / s_v, 0} of the step's tokens
  float m[kWarps][kRows], l[kWarps][kRows];
  const float4* o[kWarps];  // the warps' rows at a unit's end: [row][kD / 4], see merge_chunk
  uint64_t full[kWarps][kStages];
  int abort_flag;
  int last;
};

// Where the q-th four dims of row `row` lie in the row, while the warps merge:
// as that, the eight lanes that write (or read) at a time hit distinct banks.
__device__ __forceinline__ int merge_chunk(int row, int q) {
  return q ^ ((row >> 1) | (q >> 4 << 2));
}
static_assert(kRows * kD * 4 == kStep * kD, "a warp's rows fill a stage of K");

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte kI of two words of e4m3 values, as bf16 times 2^-120.
template <int kI>
__device__ __forceinline__ uint32_t e4m3_pair_to_bf16x2(uint32_t w0, uint32_t w1) {
  constexpr uint32_t sel = kI | (8 + kI) << 4 | (4 + kI) << 8 | (12 + kI) << 12;  // 8: the sign
  uint32_t t;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(t) : "r"(w0), "r"(w1), "n"(sel));
  return (t << 4) & 0x87f087f0u;
}
constexpr float kWeightUp = 0x1p100f, kOutUp = 0x1p20f;  // together 2^120

// Transposes an 8 x 8 matrix of 16-bit values, a row of four pairs per lane quad.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// hi = f16(x), lo = f16(kRestUp (x - hi)) of two values, packed.
constexpr float kRestUp = 0x1p11f;
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = cvt_f16x2(x0, x1);
  float h0, h1;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(h0), "=f"(h1)
      : "r"(hi));
  lo = cvt_f16x2((x0 - h0) * kRestUp, (x1 - h1) * kRestUp);
}

// Where a walk over the CTA's run of tiles stands.
struct Walk {
  int at;  // place in the line of tiles
  int seq, head, tile, ctx, n_tiles;
  int block, offset;  // where this warp's step of the tile lies in the sequence
};

__device__ __forceinline__ int clamped_ctx(const Q8Params& p, int seq) {
  return min(max(p.context_lens[seq], 0), p.max_context);
}
__device__ __forceinline__ int tiles_of(int ctx) { return max(1, (ctx + kTile - 1) / kTile); }

__device__ __forceinline__ void walk_next(const Q8Params& p, int end, Walk& w) {
  ++w.at;
  w.offset += kTile;
  while (w.offset >= p.block_size) {
    w.offset -= p.block_size;
    ++w.block;
  }
  if (++w.tile < w.n_tiles) return;
  w.at += kUnitCost;
  w.tile = 0;
  w.block = 0;
  w.offset = (threadIdx.x >> 5) * kStep;
  while (w.offset >= p.block_size) {
    w.offset -= p.block_size;
    ++w.block;
  }
  if (++w.head < p.Hkv) return;
  w.head = 0;
  ++w.seq;
  if (w.at < end) {
    w.ctx = clamped_ctx(p, w.seq);
    w.n_tiles = tiles_of(w.ctx);
  }
}

// The query rows of (seq, head) as mma operands: row g scaled by a power of two
// so that max|q| lies in [2^14, 2^15); a[k] = {first pair, second pair}, and for
// f32 queries their remainders.  (A bf16 value has 8 bits, so it is an f16 one
// down to 2^-28 of the row's largest, and below that off by 2^-39 of it.)
// Returns the factor that undoes the scaling (of row g).
template <bool kBf16>
constexpr int kQWords = kBf16 ? 2 : 4;
template <bool kBf16>
__device__ __forceinline__ float load_q(const Q8Params& p, int seq, int head, int g, int c,
                                        uint32_t (&a)[8][kQWords<kBf16>]) {
  float x[2][16];
  const bool real = g < p.G;
  const long long off = ((long long)seq * p.Hq + (long long)head * p.G + g) * kD + 16 * c;
  uint32_t big = 0;
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[hf][i] = 0.0f;
    if (real) {
      if constexpr (kBf16) {
        const uint4* src =
            reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + off + 64 * hf);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = src[i];
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[hf][8 * i + 2 * e] = bf16lo_to_f32(u[e]);
            x[hf][8 * i + 2 * e + 1] = bf16hi_to_f32(u[e]);
          }
        }
      } else {
        const float4* src =
            reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + off + 64 * hf);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 v = src[i];
          x[hf][4 * i] = v.x; x[hf][4 * i + 1] = v.y; x[hf][4 * i + 2] = v.z; x[hf][4 * i + 3] = v.w;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) big = max(big, __float_as_uint(x[hf][i]) & 0x7fffffffu);
  }
  big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
  int e = (int)(big >> 23) - 127;
  e = (big == 0 || big >= 0x7f800000u) ? 0 : max(e - 14, -126);
  const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t* f = a[4 * hf + i];
      if constexpr (kBf16) {
        f[0] = cvt_f16x2(x[hf][4 * i] * down, x[hf][4 * i + 1] * down);
        f[1] = cvt_f16x2(x[hf][4 * i + 2] * down, x[hf][4 * i + 3] * down);
      } else {
        split_f16(x[hf][4 * i] * down, x[hf][4 * i + 1] * down, f[0], f[2]);
        split_f16(x[hf][4 * i + 2] * down, x[hf][4 * i + 3] * down, f[1], f[3]);
      }
    }
  return __uint_as_float((uint32_t)(127 + e) << 23);
}

// kN consecutive dims from `d` of query row `row` of the unit.
template <bool kBf16, int kN>
__device__ __forceinline__ void write_out(const Q8Params& p, int seq, int head, int row, int d,
                                          const float (&o)[kN], float l) {
  const float f = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
  const long long i = ((long long)seq * p.Hq + (long long)head * p.G + row) * kD + d;
#pragma unroll
  for (int e = 0; e < kN; e += 2) {
    if constexpr (kBf16)
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + i + e) =
          pack_bf16x2(o[e] * f, o[e + 1] * f);
    else
      *reinterpret_cast<float2*>(static_cast<float*>(p.out) + i + e) =
          make_float2(o[e] * f, o[e + 1] * f);
  }
}

__device__ __forceinline__ void fma4(float4& o, const float4& a, float f) {
  o.x = fmaf(a.x, f, o.x);
  o.y = fmaf(a.y, f, o.y);
  o.z = fmaf(a.z, f, o.z);
  o.w = fmaf(a.w, f, o.w);
}

// Merges the partials of a unit that CTAs c0..c1 share, in CTA order.  A warp
// takes kR rows at a time, and 32 partials: a lane per partial for the factors,
// then four dimensions per lane.  kEarly partials' rows are read together with
// the factors: the launch ends with this, and each dependent read is about half
// a microsecond.
template <bool kBf16, int kR, int kEarly>
__device__ __forceinline__ void merge_parts(const Q8Params& p, int seq, int head, int c0, int c1) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r0 = warp; r0 < p.G; r0 += kWarps * kR) {
    float4 O[kR];
    float M[kR], L[kR];
#pragma unroll
    for (int x = 0; x < kR; ++x) {
      O[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      M[x] = -INFINITY;
      L[x] = 0.0f;
    }
    for (int base = c0; base <= c1; base += 32) {
      const int n = min(c1 + 1 - base, 32);
      // (the first CTA left its part in its second place: tile_split.cuh)
      const float* q = p.part + ((long long)base * 2 + (base == c0)) * kQ8PartFloats;
      const long long step = 2 * kQ8PartFloats - (base == c0 ? kQ8PartFloats : 0);
      auto at = [&](int i) {
        return i == 0 ? q : q + step + (long long)(i - 1) * 2 * kQ8PartFloats;
      };
      auto load = [&](int i, int r) {
        return __ldcg(reinterpret_cast<const float4*>(at(i) + r * kD) + lane);
      };
      float m[kR], l[kR], f[kR];
      float4 v[kR][kEarly > 0 ? kEarly : 1];
#pragma unroll
      for (int x = 0; x < kR; ++x) {
        const int r = r0 + kWarps * x;
        m[x] = -INFINITY;
        l[x] = 0.0f;
        if (r >= p.G) break;
        if (lane < n) {
          m[x] = __ldcg(at(lane) + kRows * kD + r);
          l[x] = __ldcg(at(lane) + kRows * kD + kRows + r);
        }
#pragma unroll
        for (int i = 0; i < kEarly; ++i)
          if (i < n) v[x][i] = load(i, r);
      }
#pragma unroll
      for (int x = 0; x < kR; ++x) {
        float top = fmaxf(m[x], M[x]);
#pragma unroll
        for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
        const float old = M[x] == -INFINITY ? 1.0f : fast_exp2(M[x] - top);
        f[x] = m[x] == -INFINITY ? 1.0f : fast_exp2(m[x] - top);
        float s = l[x] * f[x];
#pragma unroll
        for (int y = 16; y >= 1; y >>= 1) s += __shfl_xor_sync(0xffffffffu, s, y);
        L[x] = fmaf(L[x], old, s);
        M[x] = top;
        O[x] = make_float4(O[x].x * old, O[x].y * old, O[x].z * old, O[x].w * old);
      }
#pragma unroll
      for (int x = 0; x < kR; ++x) {
        const int r = r0 + kWarps * x;
        if (r >= p.G) break;
#pragma unroll
        for (int i = 0; i < kEarly; ++i) {
          const float fi = __shfl_sync(0xffffffffu, f[x], i);
          if (i < n) fma4(O[x], v[x][i], fi);
        }
#pragma unroll(kR > 1 ? 4 : 8)
        for (int i = kEarly; i < n; ++i)
          fma4(O[x], load(i, r), __shfl_sync(0xffffffffu, f[x], i));
      }
    }
#pragma unroll
    for (int x = 0; x < kR; ++x) {
      const int r = r0 + kWarps * x;
      if (r >= p.G) break;
      const float o[4] = {O[x].x, O[x].y, O[x].z, O[x].w};
      write_out<kBf16>(p, seq, head, r, 4 * lane, o, L[x]);
    }
  }
}

template <bool kBf16, int kCtas>  // kCtas: CTAs per SM
__global__ void __launch_bounds__(kThreads, kCtas)
    decode_q8_kernel(const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, Q8Params p) {
  extern __shared__ uint8_t smem_raw[];
  Q8Smem& sm = *reinterpret_cast<Q8Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_barrier_init();
  }
  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    sm.last = timeout_recorded(p.status);  // then: skip the work
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  volatile int* abort_flag = &sm.abort_flag;
  const tilesplit::Run run =
      tilesplit::find_run(p.n_seqs, blockIdx.x, gridDim.x, 1, [&](int s) {
        return tilesplit::SeqTiles{p.Hkv, tiles_of(clamped_ctx(p, s)) + kUnitCost};
      });
  __syncthreads();
  if (run.begin >= run.end || sm.last) return;

  Walk w;
  w.at = run.begin;
  w.seq = run.seq;
  w.ctx = clamped_ctx(p, w.seq);
  w.n_tiles = tiles_of(w.ctx);
  w.head = (run.begin - run.seq_first) / (w.n_tiles + kUnitCost);
  w.tile = (run.begin - run.seq_first) % (w.n_tiles + kUnitCost) - kUnitCost;
  if (w.tile < 0) {  // the run begins before a unit's first tile
    w.at -= w.tile;
    w.tile = 0;
    if (w.at >= run.end) return;
  }
  w.block = (w.tile * kTile + warp * kStep) / p.block_size;
  w.offset = (w.tile * kTile + warp * kStep) % p.block_size;

  // ---- loads: one step = this warp's 32 tokens of a tile ----
  Walk ahead = w;
  int issued = 0, used = 0;
  const uint64_t policy = l2_policy_evict_first();
  auto block_of = [&](const Walk& x) -> int {
    const int t0 = x.tile * kTile + warp * kStep;
    if (x.at >= run.end || t0 >= x.ctx) return 0;
    return p.block_tables[(long long)x.seq * p.max_blocks + x.block];
  };
  int next_bid = block_of(ahead);
  auto issue = [&]() {  // the step at `ahead`, if it has tokens; moves `ahead` on
    const int t0 = ahead.tile * kTile + warp * kStep;
    const bool some = t0 < ahead.ctx;
    long long bid = next_bid;
    const int head = ahead.head, offset = ahead.offset;
    const int seq = ahead.seq, raw = ahead.tile == 0 && ahead.head == 0;
    walk_next(p, run.end, ahead);
    next_bid = block_of(ahead);  // used a step later: its latency is off the path
    if (raw && warp == 0 && lane == 0) {
      const int ctx = p.context_lens[seq];
      if (ctx < 0 || ctx > p.max_context)
        record_error(p.status, NVATTN_ERR_OUT_OF_RANGE, 91, ctx);
    }
    if (!some) return;
    if (lane == 0) {
      if (bid < 0 || bid >= p.num_blocks) {
        record_error(p.status, NVATTN_ERR_OUT_OF_RANGE, 92, bid);
        bid = 0;  // keep the ring in step; the result is flagged
      }
      const int st = issued % kStages;
      uint64_t* bar = &sm.full[warp][st];
      const int page = (int)((long long)p.layer * p.num_blocks + bid);
      const int row = head * p.block_size + offset;
      const long long srow = (long long)page * p.Hkv * p.block_size + row;
      mbar_arrive_expect_tx(bar, 2 * kStep * (kD + 4));
      tma_load_3d_hint(sm.ring[warp].k[st], &tm_k, bar, 0, row, page, policy);
      tma_load_3d_hint(sm.ring[warp].v[st], &tm_v, bar, 0, row, page, policy);
      bulk_load(sm.ks[warp][st], p.k_scale + srow, kStep * 4, bar, policy);
      bulk_load(sm.vs[warp][st], p.v_scale + srow, kStep * 4, bar, policy);
    }
    ++issued;
  };
  // (`ahead` may run past the last tile by the ring's depth: no step there)
  for (int i = 0; i < kStages && ahead.at < run.end; ++i) issue();

  uint32_t qa[8][kQWords<kBf16>];
  float o[8][4];  // [j]: dims 16 ch + 2 j (elements 0, 1: rows 2c, 2c + 1) and 2 j + 1 (2, 3)
  const int pr = (g >> 1) | ((g & 1) << 2);

  while (w.at < run.end) {
    // ---- one unit's part of the run ----
    const int seq = w.seq, head = w.head, first = w.tile, n_tiles = w.n_tiles, ctx = w.ctx;
    const int unit0 = w.at - w.tile;
    const float up_g = load_q<kBf16>(p, seq, head, g, c, qa);
    // the lane's query rows from here on: 2c and 2c + 1
    const float up[2] = {__shfl_sync(0xffffffffu, up_g, 8 * c),
                         __shfl_sync(0xffffffffu, up_g, 8 * c + 4)};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;

    int done = 0;  // tiles of the unit in this run
    do {
      const int t0 = w.tile * kTile + warp * kStep;
      if (t0 < ctx) {
        const int st = used % kStages;
        mbar_wait(&sm.full[warp][st], (used / kStages) & 1, p.status, abort_flag, 93);
        ++used;
        uint8_t* kt = sm.ring[warp].k[st];
        uint8_t* vt = sm.ring[warp].v[st];
        const int n = min(ctx - t0, kStep);
        // ---- the tokens' factors ----
        {
          const float sk = sm.ks[warp][st][lane], sv = sm.vs[warp][st][lane];
          // A NaN scale (a row that held a NaN or an infinity) stays NaN; a scale
          // of 0 (a row never written in a cache that began as zeros) counts as the
          // least one, 2^-100: its reciprocal would be 2^127, two of which overflow.
          const uint32_t e = max(__float_as_uint(sv) >> 23, 27u);
          float4 f = make_float4(sk * p.scale_log2, (float)((int)e - 127) + (sv - sv),
                                 __uint_as_float((254u - e) << 23), 0.0f);
          if (lane >= n) {
            // Slots behind the context hold anything: weight zero, and rows
            // of zeros so that no NaN meets it.
            f = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
            const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              reinterpret_cast<uint4*>(kt + lane * kD)[i] = z;
              reinterpret_cast<uint4*>(vt + lane * kD)[i] = z;
            }
          }
          if (n < kStep) fence_proxy_async_smem();  // before the ring's next copy into this stage
          sm.tok[warp][lane] = f;
          __syncwarp();
        }
        // ---- scores: two tiles of 16 tokens (rows g and g + 8 of the lane) ----
        float s[2][2][4];  // [tile][product with the queries, with their remainders]
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mt][0][e] = s[mt][1][e] = 0.0f;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t u[4][4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint4 v = *reinterpret_cast<const uint4*>(kt + (8 * t + pr) * kD +
                                                            (((c + 4 * hf) ^ pr) << 4));
            u[t][0] = v.x; u[t][1] = v.y; u[t][2] = v.z; u[t][3] = v.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              const uint32_t a[4] = {e4m3x2_to_f16x2(u[2 * mt][i] & 0xffffu),
                                     e4m3x2_to_f16x2(u[2 * mt + 1][i] & 0xffffu),
                                     e4m3x2_to_f16x2(u[2 * mt][i] >> 16),
                                     e4m3x2_to_f16x2(u[2 * mt + 1][i] >> 16)};
              const uint32_t* q = qa[4 * hf + i];
              mma_f16(s[mt][0], a, q[0], q[1]);
              if constexpr (!kBf16) mma_f16(s[mt][1], a, q[2], q[3]);
            }
        }
        float x[4][2], inv[4];  // [eight tokens][query row]
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float4 f = sm.tok[warp][8 * t + pr];
          const int mt = t >> 1, e = 2 * (t & 1);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float y = s[mt][0][e + r];
            if constexpr (!kBf16) y = fmaf(s[mt][1][e + r], 1.0f / kRestUp, y);
            x[t][r] = fmaf(y * up[r], f.x, f.y);
          }
          inv[t] = f.z;
        }
        float top[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) top[r] = fmax3(x[0][r], x[1][r], fmaxf(x[2][r], x[3][r]));
        if (__any_sync(0xffffffffu, top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
          // (rare after the first step: the reference moves in strides of 2^8)
          float alpha[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int lanes = 4; lanes < 32; lanes *= 2)
              top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], lanes));
            const float m_new = top[r] > m[r] + kSlack ? top[r] : m[r];
            alpha[r] = m_new == m[r] ? 1.0f : fast_exp2(m[r] - m_new);
            m[r] = m_new;
            l[r] *= alpha[r];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] *= alpha[e & 1];
        }
        uint32_t wb[4][3];  // [eight tokens][term of the weights], as operands
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          // (a step has a key: m is -inf only where every key's score is NaN)
          float w0 = fast_exp2(x[t][0] - m[0]), w1 = fast_exp2(x[t][1] - m[1]);
          l[0] = fmaf(w0, inv[t], l[0]);
          l[1] = fmaf(w1, inv[t], l[1]);
          w0 *= kWeightUp;
          w1 *= kWeightUp;
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            uint32_t term;
            split_term(w0, w1, term);
            wb[t][i] = transpose8x8(term);
          }
        }
        // ---- o += V8 w ----
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t v[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 16 * ks + c + 4 * i;
            const uint4 t = *reinterpret_cast<const uint4*>(vt + r * kD + ((pr ^ (r & 7)) << 4));
            v[i][0] = t.x; v[i][1] = t.y; v[i][2] = t.z; v[i][3] = t.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[2][4] = {{e4m3_pair_to_bf16x2<0>(v[0][i], v[1][i]),
                                       e4m3_pair_to_bf16x2<1>(v[0][i], v[1][i]),
                                       e4m3_pair_to_bf16x2<0>(v[2][i], v[3][i]),
                                       e4m3_pair_to_bf16x2<1>(v[2][i], v[3][i])},
                                      {e4m3_pair_to_bf16x2<2>(v[0][i], v[1][i]),
                                       e4m3_pair_to_bf16x2<3>(v[0][i], v[1][i]),
                                       e4m3_pair_to_bf16x2<2>(v[2][i], v[3][i]),
                                       e4m3_pair_to_bf16x2<3>(v[2][i], v[3][i])}};
#pragma unroll
            for (int term = 2; term >= 0; --term)  // the small terms first
#pragma unroll
              for (int h = 0; h < 2; ++h)
                mma_bf16(o[2 * i + h], a[h], wb[2 * ks][term], wb[2 * ks + 1][term]);
          }
        }
        __syncwarp();  // every lane has read the stage
      }
      walk_next(p, run.end, w);
      ++done;
      if (w.at >= run.end || w.tile == 0) break;  // the unit's last: issued after the merge
      if (ahead.at < run.end) issue();
    } while (true);

    // ---- merge the warps ----
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int lanes = 4; lanes < 32; lanes *= 2)
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], lanes);
      if (g == 0) {
        sm.m[warp][2 * c + r] = m[r];
        sm.l[warp][2 * c + r] = l[r];
      }
    }
    const bool whole = first == 0 && done == n_tiles;
    float* part = p.part + ((long long)blockIdx.x * 2 + (first == 0 ? 1 : 0)) * kQ8PartFloats;
    // The warp's rows go to the K part of the stage that is filled next (free:
    // the last tile's load has not been issued); a warp then merges two rows.
    float4* rows = reinterpret_cast<float4*>(sm.ring[warp].k[issued % kStages]);
    if (lane == 0) sm.o[warp] = rows;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        rows[(2 * c + r) * (kD / 4) + merge_chunk(2 * c + r, 4 * pr + j)] =
            make_float4(o[2 * j][r] * kOutUp, o[2 * j][2 + r] * kOutUp,
                        o[2 * j + 1][r] * kOutUp, o[2 * j + 1][2 + r] * kOutUp);
    __syncthreads();
    for (int r = warp; r < p.G; r += kWarps) {
      float M = -INFINITY, L = 0.0f;
      float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) M = fmaxf(M, sm.m[i][r]);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float f = sm.m[i][r] == -INFINITY ? 1.0f : fast_exp2(sm.m[i][r] - M);
        fma4(O, sm.o[i][r * (kD / 4) + merge_chunk(r, lane)], f);
        L = fmaf(sm.l[i][r], f, L);
      }
      if (whole) {
        const float y[4] = {O.x, O.y, O.z, O.w};
        write_out<kBf16>(p, seq, head, r, 4 * lane, y, L);
      } else {
        *reinterpret_cast<float4*>(part + r * kD + 4 * lane) = O;
        if (lane == 0) {
          part[kRows * kD + r] = M;
          part[kRows * kD + kRows + r] = L;
        }
      }
    }
    fence_proxy_async_smem();  // before the next copy into the stage
    __syncthreads();           // the rows have been read
    if (ahead.at < run.end) issue();
    if (!whole) {
      const int c0 = unit0 / run.per, c1 = (unit0 + n_tiles - 1) / run.per;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int last = atomicAdd(p.tickets + c0, 1) == c1 - c0;
        if (last) atomicExch(p.tickets + c0, 0);  // re-armed for the next launch
        sm.last = last;
      }
      __syncthreads();
      if (sm.last) {
        __threadfence();
        if constexpr (kCtas == 2)
          merge_parts<kBf16, 2, 4>(p, seq, head, c0, c1);
        else  // (three CTAs per SM have no registers for that)
          merge_parts<kBf16, 1, 0>(p, seq, head, c0, c1);
      }
      __syncthreads();  // sm.last is free
    }
  }
  // After a wait that ran out, copies may still be in flight: wait (bounded)
  // for the ring's last ones before the CTA's shared memory goes away.
  if (*abort_flag && lane == 0)
    for (int i = max(0, issued - kStages); i < issued; ++i)
      mbar_wait(&sm.full[warp][i % kStages], (i / kStages) & 1, p.status, 94);
}

}  // namespace

nvattn_status launch_paged_decode_q8(nvattn_handle* h, int layer, int n_seqs, const void* q,
                                     nvattn_dtype dtype, const uint8_t* k_q8,
                                     const float* k_scale, const uint8_t* v_q8,
                                     const float* v_scale, const int32_t* block_tables,
                                     int max_blocks, const int32_t* context_lens,
                                     int max_context_len, void* out, cudaStream_t stream) {
  if (n_seqs == 0) return NVATTN_OK;
  CUtensorMap tk, tv;
  nvattn_status st = get_q8_tensor_map(h, k_q8, kStep, &tk);
  if (st != NVATTN_OK) return st;
  st = get_q8_tensor_map(h, v_q8, kStep, &tv);
  if (st != NVATTN_OK) return st;
  Q8Params p = {};
  p.Hq = h->cfg.n_q_heads;
  p.Hkv = h->cfg.n_kv_heads;
  p.G = p.Hq / p.Hkv;
  p.layer = layer;
  p.block_size = h->cfg.block_size;
  p.max_blocks = max_blocks;
  p.n_seqs = n_seqs;
  p.max_context = max_context_len;
  p.num_blocks = h->cfg.num_blocks;
  p.scale_log2 = h->cfg.scale * kLog2e;
  p.q = q;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.out = out;
  p.part = h->ws_part;
  p.tickets = h->part_tickets;
  p.status = h->status_dev;
  const long long tiles = (long long)n_seqs * p.Hkv * ((max_context_len + kTile - 1) / kTile);
  if (tiles + (long long)n_seqs * p.Hkv * (1 + kUnitCost) >= tilesplit::kMaxPlaces)
    return NVATTN_ERR_UNSUPPORTED;
  const int per_sm = tiles >= (long long)kFullGridTiles * kQ8CtasPerSm * h->sm_count
                         ? kQ8CtasPerSm : kQ8CtasPerSm - 1;
  using Kernel = void (*)(const CUtensorMap, const CUtensorMap, Q8Params);
  constexpr size_t smem_full = sizeof(Q8Smem) + 1024;
  static_assert(kQ8CtasPerSm == 3 && 3 * (smem_full + 1024) <= 228 * 1024, "three per SM");
  static_assert(smem_full <= kTwoCtaSmem && 2 * (kTwoCtaSmem + 1024) <= 228 * 1024, "two per SM");
  const bool bf16 = dtype == NVATTN_DTYPE_BF16, full = per_sm == kQ8CtasPerSm;
  const Kernel kernels[2][2] = {{decode_q8_kernel<false, 2>, decode_q8_kernel<false, 3>},
                                {decode_q8_kernel<true, 2>, decode_q8_kernel<true, 3>}};
  // (atomic: handles on different threads may launch at the same time)
  static std::atomic<unsigned long long> attr_set_mask{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return NVATTN_ERR_CUDA;
  if (dev >= 64 || !(attr_set_mask.load(std::memory_order_relaxed) & (1ull << dev))) {
    for (int i = 0; i < 4; ++i)
      if (cudaFuncSetAttribute(kernels[i >> 1][i & 1], cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)((i & 1) ? smem_full : kTwoCtaSmem)) != cudaSuccess)
        return NVATTN_ERR_CUDA;
    if (dev < 64) attr_set_mask.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  kernels[bf16][full]<<<per_sm * h->sm_count, kThreads, full ? smem_full : kTwoCtaSmem,
                        stream>>>(tk, tv, p);
  return cudaGetLastError() == cudaSuccess ? NVATTN_OK : NVATTN_ERR_CUDA;
}

}  // namespace nvattn
