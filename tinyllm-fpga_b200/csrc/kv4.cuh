// kv4.cuh -- the 4-bit paged KV cache: record layout, tile arithmetic, batch
// description shared by kv4.cu (rope, append, read), kv4_attn.cu and
// kv4_prompt.cu (attention).
//
// Number format.  The framework's tiles of 16 elements with one exponent
// (tile_quantize, gen_smollm_blockfp_full.py:90-97), with 4-bit mantissas:
//   e = clip(floor(log2(max|v|)) + 1, -17, 12)
//   m = clip(rint(v * 2^(3 - e)), -8, 7),   value = m * 2^(e - 3)
// held as the nibble m + 8 and the byte B = e + 18 in 1..30, so value =
// (nibble - 8) * 2^(B - 21).  The exponent window makes every value exact in
// bfloat16, and 2^-4 times it exact in binary16 (quanta 2^-24 .. 2^5, where
// 1032 * 2^5 still fits), so both tensor-core types hold the cache without a
// further rounding.  |v| > 3584 saturates.
//
// Record of one (page, KV head), page * HD * 9 / 8 bytes:
//   keys    [page/4][HD/8][4 positions][4 B]      nibble n = dim 8 u + n
//   values  [page/8][HD/4][4 i][2 h][2 B]         position 8 o + 4 h + i, nibble n = dim 4 u + n
//   key exponents [HD/16][page], value exponents [HD/16][page]
// A key word holds 8 dims of one position, and in 16-bit halves the dim pairs
// (n, n + 4): the pairs of a tensor-core operand whose contraction axis is
// the head dim.  A value word holds 4 dims of the positions i and i + 4: the
// pairs of an operand whose contraction axis is the position.  No two
// positions share a byte, so tokens of one page may be written concurrently.
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/bfp200.h"

namespace bfp {
namespace kv4 {

constexpr int E_MIN = -17, E_MAX = 12;

// The batch as the kernels see it (pointers on the device).
struct Batch {
  uint8_t* pool;
  const int* bt;          // [n_seq][bt_ld]: page of every `page` positions
  const int* q_start;     // [n_seq + 1]: this call's tokens of each sequence
  const int* lens;        // [n_seq]: positions of each sequence, this call's included
  int n_pages, page, page_shift, H, n_seq, max_pages, T;
  long long bt_ld;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// VE consecutive elements, as 16-byte words when ALIGNED; by the read-only path
// (NC) where nothing is written in place.
template <typename T, int VE, bool ALIGNED, bool NC>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[VE]) {
  if constexpr (ALIGNED) {
    constexpr int NW = VE * (int)sizeof(T) / 16;
    alignas(16) T v[VE];
    #pragma unroll
    for (int i = 0; i < NW; ++i) reinterpret_cast<uint4*>(v)[i] = NC ? __ldg(reinterpret_cast<const uint4*>(p) + i) : reinterpret_cast<const uint4*>(p)[i];
    #pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = to_f(v[i]);
  } else {
    #pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = to_f(p[i]);
  }
}
template <typename T, int VE, bool ALIGNED>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VE]) {
  alignas(16) T v[VE];
  #pragma unroll
  for (int i = 0; i < VE; ++i) v[i] = from_f<T>(f[i]);
  if constexpr (ALIGNED) {
    constexpr int NW = VE * (int)sizeof(T) / 16;
    #pragma unroll
    for (int i = 0; i < NW; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
  } else {
    #pragma unroll
    for (int i = 0; i < VE; ++i) p[i] = v[i];
  }
}

// Tile exponent from the bits of max|v|: floor(log2) + 1 of a normal number
// is its exponent field - 126; subnormals and 0 clip to E_MIN, Inf to E_MAX.
__device__ __forceinline__ int tile_e(float top) {
  const int e = (int)(__float_as_uint(top) >> 23) - 126;
  return min(max(e, E_MIN), E_MAX);
}
// Mantissa of v at tile exponent e (up = 2^(3 - e)).  The product with a power of two is exact
// where it matters (an underflowing one rounds to 0 anyway); the conversion
// rounds half to even, saturates +-Inf and takes NaN to 0.
__device__ __forceinline__ int mantissa(float v, float up) { return min(max(__float2int_rn(__fmul_rn(v, up)), -8), 7); }
__device__ __forceinline__ float pow2f(int k) { return __int_as_float((k + 127) << 23); }

// The sequence whose tokens contain token t: the last b with q_start[b] <= t.
// One warp narrows the range 32-fold per load.
__device__ __forceinline__ int find_seq(const int* q_start, int n_seq, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = n_seq;                      // answer in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) >> 5;
    const int at = lo + lane * step;
    const bool le = at < lo + n && __ldg(q_start + at) <= t;
    const int k = max(__popc(__ballot_sync(0xffffffffu, le)) - 1, 0);
    n = min(step, n - k * step);
    lo += k * step;
  }
  return lo;
}

// Dynamic shared memory of a kernel on the current device, raised once.
template <typename K>
cudaError_t allow_smem(K* kern, size_t bytes, std::atomic<unsigned char> (&done)[128]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || done[dev].load(std::memory_order_relaxed)) return e;   // (device_ready keeps dev below 128)
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done[dev].store(1, std::memory_order_relaxed);
  return e;
}

int fill_batch(const bfp200_kv4_batch& in, Batch* out, const char* who);   // BFP200_OK or the error of the calling thread
int device_ready(const char* who, int* n_sm);

}  // namespace kv4
}  // namespace bfp
