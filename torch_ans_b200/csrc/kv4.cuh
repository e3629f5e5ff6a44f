// kv4.cuh -- layout and arithmetic of the 4-bit key/value cache shared by its kernels.
//
// The cache is codes[num_pages][2][kv_heads][page_size][head_dim / 2] and, beside it,
// params[num_pages][2][kv_heads][page_size] of (scale, offset) in bfloat16; a code c stands for
// c * scale + offset.  c has 4 significant bits and scale 8, so c * scale is exact in float and the
// value takes one rounding whether or not the compiler fuses the product and the sum.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/torch_ans_b200.h"

namespace tans {
namespace kv4 {

// Division by a number that the host knows: floor(n / d) for n < 2^31 is mulhi(2 n, m) >> l with
// l = ceil(log2 d), m = ceil(2^(31 + l) / d) (Granlund and Montgomery).
struct Divider {
  uint32_t d, m, l;
  static Divider of(uint32_t d) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    return {d, (uint32_t)(((1ull << (31 + l)) + d - 1) / d), l};
  }
  __device__ __forceinline__ int div(int n) const { return (int)(__umulhi(2u * (uint32_t)n, m) >> l); }
};

struct Pool {
  const uint8_t* codes;
  const uint32_t* params;  // (scale, offset): low and high half
  int64_t num_pages;
  int kv_heads, page_size, head_dim;

  // first row of a page's side and head, in rows
  __host__ __device__ int64_t row(int64_t page, int side, int head) const {
    return ((page * 2 + side) * kv_heads + head) * (int64_t)page_size;
  }
};

// the scale and the offset are the two bfloat16 halves of one word
__device__ __forceinline__ float scale_of(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float offset_of(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

template <typename T>
struct Half2;
template <>
struct Half2<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Half2<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};

inline bool pool_ok(const void* codes, const void* params, int64_t num_pages, int kv_heads, int page_size,
                    int head_dim) {
  if (num_pages < 0 || kv_heads < 1 || kv_heads > 65535 || page_size < 16 || page_size > (1 << 20) ||
      page_size % 16 != 0 || (int64_t)kv_heads * page_size >= ((int64_t)1 << 30))
    return false;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return false;
  if (num_pages > 0 && (!codes || !params)) return false;
  // rows are read 16 bytes at a time
  return (reinterpret_cast<uintptr_t>(codes) & 15) == 0 && (reinterpret_cast<uintptr_t>(params) & 15) == 0;
}

}  // namespace kv4
}  // namespace tans
