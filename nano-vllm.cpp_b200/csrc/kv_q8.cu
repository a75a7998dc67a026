// kv_q8.cu -- reading rows of the 8-bit paged KV cache back as bf16, f16 or
// f32 rows (the store that writes them is kv_store.cu's).
//
// value = e4m3 payload * 2^E.  e4m3 widens to f16 exactly, the product with a
// power of two is exact in f32, and bf16 holds it exactly (4 significant
// bits); f16 rounds to nearest even and overflows above 65504.
//
// Bound by memory: per row 132 bytes in, 128 elements out.  Eight lanes own a
// row (16 payload bytes each, so a row leaves as whole 32-byte sectors), and
// each lane has kUnroll independent rows in flight (65,536 tokens x 8 kv heads
// to bf16: 71.8 us with two, 5.7 TB/s, 89 % of the measured copy rate; 77.9 us
// with one, 74.2 with four, 88.6 with eight); blockIdx.y is K or V.
#include "common.cuh"
#include "internal.h"

namespace nvattn {
namespace {

constexpr int kD = 128;
constexpr int kThreads = 256;
constexpr int kUnroll = 2;
constexpr int kRowsPerPass = kThreads / 8;

struct LoadParams {
  int rows;  // n_tokens * Hkv
  int Hkv, layer, block_size;
  long long n_slots, num_blocks;
  const int32_t* slots;
  const uint8_t *k_q8, *v_q8;
  const float *k_scale, *v_scale;
  void *k_out, *v_out;
  DeviceStatus* status;
};

template <typename T>
__device__ __forceinline__ void write16(T* dst, const float (&y)[16]);

template <>
__device__ __forceinline__ void write16<float>(float* dst, const float (&y)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<float4*>(dst)[i] =
        make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
}

struct Bf16 { uint16_t v; };
struct F16 { uint16_t v; };

template <>
__device__ __forceinline__ void write16<Bf16>(Bf16* dst, const float (&y)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    reinterpret_cast<uint4*>(dst)[i] =
        make_uint4(cvt_bf16x2(y[8 * i], y[8 * i + 1]), cvt_bf16x2(y[8 * i + 2], y[8 * i + 3]),
                   cvt_bf16x2(y[8 * i + 4], y[8 * i + 5]), cvt_bf16x2(y[8 * i + 6], y[8 * i + 7]));
}

template <>
__device__ __forceinline__ void write16<F16>(F16* dst, const float (&y)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    reinterpret_cast<uint4*>(dst)[i] =
        make_uint4(cvt_f16x2(y[8 * i], y[8 * i + 1]), cvt_f16x2(y[8 * i + 2], y[8 * i + 3]),
                   cvt_f16x2(y[8 * i + 4], y[8 * i + 5]), cvt_f16x2(y[8 * i + 6], y[8 * i + 7]));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kv_load_q8_kernel(LoadParams p) {
  const bool is_v = blockIdx.y != 0;
  const uint8_t* q8 = is_v ? p.v_q8 : p.k_q8;
  const float* scale = is_v ? p.v_scale : p.k_scale;
  T* out = static_cast<T*>(is_v ? p.v_out : p.k_out);
  const int l8 = threadIdx.x & 7;
  const long long row0 = (long long)blockIdx.x * (kRowsPerPass * kUnroll) + (threadIdx.x >> 3);
  uint4 w[kUnroll];
  float sc[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long long r = row0 + u * kRowsPerPass;
    w[u] = make_uint4(0, 0, 0, 0);  // a padding row, or a slot outside the cache: zeros
    sc[u] = 0.0f;
    if (r < p.rows) {
      const int t = (int)((unsigned)r / (unsigned)p.Hkv), head = (int)r - t * p.Hkv;
      const int slot = p.slots[t];
      if (slot >= 0 && (long long)slot < p.n_slots) {
        const long long row = (((long long)p.layer * p.num_blocks + slot / p.block_size) * p.Hkv +
                               head) * p.block_size + slot % p.block_size;
        w[u] = __ldcs(reinterpret_cast<const uint4*>(q8 + row * kD + 16 * l8));
        sc[u] = scale[row];
      } else if (slot >= 0 && l8 == 0) {
        record_error(p.status, NVATTN_ERR_OUT_OF_RANGE, 90, slot);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long long r = row0 + u * kRowsPerPass;
    if (r < p.rows) {
      float y[16], f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e4m3x4_to_f32(i == 0 ? w[u].x : i == 1 ? w[u].y : i == 2 ? w[u].z : w[u].w, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * i + e] = f[e] * sc[u];
      }
      write16(out + r * kD + 16 * l8, y);
    }
  }
}

}  // namespace

nvattn_status launch_kv_load_q8(nvattn_handle* h, int layer, int n_tokens, const int32_t* slots,
                                const uint8_t* k_q8, const float* k_scale, const uint8_t* v_q8,
                                const float* v_scale, nvattn_dtype out_dtype, void* k_out,
                                void* v_out, cudaStream_t stream) {
  if (n_tokens == 0) return NVATTN_OK;
  const long long rows = (long long)n_tokens * h->cfg.n_kv_heads;
  if (rows > 0x7fffffffLL) return NVATTN_ERR_INVALID_ARG;
  LoadParams p = {};
  p.rows = (int)rows;
  p.Hkv = h->cfg.n_kv_heads;
  p.layer = layer;
  p.block_size = h->cfg.block_size;
  p.n_slots = h->n_slots;
  p.num_blocks = h->cfg.num_blocks;
  p.slots = slots;
  p.k_q8 = k_q8;
  p.v_q8 = v_q8;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.k_out = k_out;
  p.v_out = v_out;
  p.status = h->status_dev;
  const int per_block = kRowsPerPass * kUnroll;
  const dim3 grid((unsigned)((rows + per_block - 1) / per_block), 2);
  switch (out_dtype) {
    case NVATTN_DTYPE_BF16: kv_load_q8_kernel<Bf16><<<grid, kThreads, 0, stream>>>(p); break;
    case NVATTN_DTYPE_F16: kv_load_q8_kernel<F16><<<grid, kThreads, 0, stream>>>(p); break;
    default: kv_load_q8_kernel<float><<<grid, kThreads, 0, stream>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? NVATTN_OK : NVATTN_ERR_CUDA;
}

}  // namespace nvattn
