// kv4_store.cu -- writing and reading the 4-bit key/value cache: append (rotation, quantisation),
// gather (values) and the exchange of pages with the entropy coder's symbols.
#include <cuda_runtime.h>

#include "kv4.cuh"
#include "launch.cuh"
#include "rans_host.h"

namespace tans {
namespace kv4 {
namespace {

constexpr int kThreads = 256;
constexpr float kTinyScale = 7.8886090522101181e-31f;  // 2^-100

// the smaller / larger of two floats, NaN if either is
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct AppendArgs {
  uint8_t* codes;
  uint32_t* params;
  Pool pool;
  const void *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  void* q_out;
  int q_heads;
  const int64_t* slots;
  int64_t tokens;
  const float* rotation;
  int64_t rotation_rows;
  int rotary;
  const int64_t* positions;
  uint32_t* status;
};

// 8 consecutive elements of a row, as they are
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load8(const T* p) {
  if constexpr (VEC) return *reinterpret_cast<const uint4*>(p);
  const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
  return make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16,
                    u[6] | (uint32_t)u[7] << 16);
}
template <typename T>
__device__ __forceinline__ void floats(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Half2<T>::unpack(u[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Rotation and quantisation, head_dim / 8 lanes for each row (one token's head), 8 channels a lane; a
// group of lanes takes ROWS rows of one token, so that the token's cosines and sines are read once for
// all of them and the loads of the rows do not wait for one another.
//
// What it may not do without is bytes: 2 read and 2 written for a query's channel, 2 read and about 0.53
// written for a key's or a value's.  16,381 tokens of 32 + 16 heads of 128 (355 MB): see the table of
// measurements for the time.  The products and sums of the rotation are rounded one by one (no fused
// multiply-add), so the codes do not depend on the compiler's choices.
//
// The quotient (x - offset) / scale is the correctly rounded one, so that ties (common: x has 8 or 11
// bits, scale 8) go to the even code; it takes one division a row and, by Markstein's theorem, two fused
// steps a channel: with y the correctly rounded 1 / scale and q0 = d y, q0 + (d - q0 scale) y rounds
// correctly.
template <int D, typename T, bool VEC, bool INTERLEAVED, int ROWS>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x % L, d0 = lane * 8;
  const int per_token = a.q_heads + 2 * a.pool.kv_heads, chunks = (per_token + ROWS - 1) / ROWS;
  const int64_t group = blockIdx.x * (int64_t)(kThreads / L) + threadIdx.x / L;
  const int64_t token = min(group / chunks, a.tokens - 1);  // groups past the end keep the warp's shuffles whole
  const int r0 = (int)(group % chunks) * ROWS;
  const int rows = group >= a.tokens * chunks ? 0 : min(ROWS, per_token - r0);

  auto source = [&](int r) -> const T* {  // row r of the token: queries, keys, values
    if (r < a.q_heads) return static_cast<const T*>(a.q) + token * a.q_ts + r * a.q_hs;
    r -= a.q_heads;
    if (r < a.pool.kv_heads) return static_cast<const T*>(a.k) + token * a.k_ts + r * a.k_hs;
    return static_cast<const T*>(a.v) + token * a.v_ts + (r - a.pool.kv_heads) * a.v_hs;
  };
  uint4 raw[ROWS];
#pragma unroll
  for (int n = 0; n < ROWS; ++n) raw[n] = n < rows ? load8<T, VEC>(source(r0 + n) + d0) : make_uint4(0, 0, 0, 0);

  const int64_t slot = r0 + rows > a.q_heads ? a.slots[token] : -1;
  bool known = false;
  float c[8], s[8];
  const int half = a.rotary / 2;
  const bool first = d0 < half;
  if (a.rotary > 0) {
    const int64_t pos = a.positions[token];
    known = pos >= 0 && pos < a.rotation_rows;
    if (!known && a.status && lane == 0 && r0 == 0 && rows > 0) atomicOr(a.status, TANS_DEV_BAD_INDEX);
    if (known && d0 < a.rotary) {
      const float* cosines = a.rotation + pos * a.rotary + (INTERLEAVED ? d0 / 2 : (first ? d0 : d0 - half));
#pragma unroll
      for (int i = 0; i < (INTERLEAVED ? 4 : 8); i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(cosines + i), y = *reinterpret_cast<const float4*>(cosines + half + i);
        c[i] = x.x; c[i + 1] = x.y; c[i + 2] = x.z; c[i + 3] = x.w;
        s[i] = y.x; s[i + 1] = y.y; s[i + 2] = y.z; s[i + 3] = y.w;
      }
    }
  }
  const bool turns = known && d0 < a.rotary;
  bool stores = slot >= 0;
  if (slot >= a.pool.num_pages * a.pool.page_size) {
    stores = false;
    if (a.status && lane == 0) atomicOr(a.status, TANS_DEV_BAD_INDEX);
  }
  const int64_t page = stores ? slot / a.pool.page_size : 0;
  const int in_page = stores ? (int)(slot - page * a.pool.page_size) : 0;

#pragma unroll
  for (int n = 0; n < ROWS; ++n) {
    const int r = r0 + n;
    const bool live = n < rows, query = r < a.q_heads, value = r >= a.q_heads + a.pool.kv_heads;
    float x[8];
    floats<T>(raw[n], x);
    if constexpr (INTERLEAVED) {
      if (turns && !value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[2 * i], w = x[2 * i + 1];
          x[2 * i] = __fsub_rn(__fmul_rn(u, c[i]), __fmul_rn(w, s[i]));
          x[2 * i + 1] = __fadd_rn(__fmul_rn(w, c[i]), __fmul_rn(u, s[i]));
        }
      }
    } else if (a.rotary > 0) {
      // the partner channels are half / 8 lanes away
      const int warp_lane = threadIdx.x & 31;
      const int partner = d0 < a.rotary ? (first ? warp_lane + half / 8 : warp_lane - half / 8) : warp_lane;
      uint4 w;
      w.x = __shfl_sync(0xffffffffu, raw[n].x, partner);
      w.y = __shfl_sync(0xffffffffu, raw[n].y, partner);
      w.z = __shfl_sync(0xffffffffu, raw[n].z, partner);
      w.w = __shfl_sync(0xffffffffu, raw[n].w, partner);
      if (turns && !value) {
        float y[8];
        floats<T>(w, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xc = __fmul_rn(x[i], c[i]), ys = __fmul_rn(y[i], s[i]);
          x[i] = first ? __fsub_rn(xc, ys) : __fadd_rn(xc, ys);
        }
      }
    }
    if (query && live) {
      uint4 w;
      w.x = Half2<T>::pack(x[0], x[1]);
      w.y = Half2<T>::pack(x[2], x[3]);
      w.z = Half2<T>::pack(x[4], x[5]);
      w.w = Half2<T>::pack(x[6], x[7]);
      *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + (token * a.q_heads + r) * D + d0) = w;
    }
    if (__all_sync(0xffffffffu, query || !live || !stores)) continue;

    // the row's range, then its codes
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = min_nan(lo, x[i]);
      hi = max_nan(hi, x[i]);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (query || !live || !stores) continue;
    const float offset = __bfloat162float(__float2bfloat16_rn(lo));
    // the product with the float nearest 1/15 is the quotient up to a unit in float's last place, 2^-15
    // of one in bfloat16's
    float scale = __bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, offset), 1.0f / 15.0f)));
    if (scale < kTinyScale) scale = 0.0f;
    const bool finite = isfinite(scale) && isfinite(offset);
    uint32_t packed = 0;
    if (finite && scale > 0.0f) {
      const float y = __frcp_rn(scale);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = __fsub_rn(x[i], offset), q0 = __fmul_rn(d, y);
        const float q = __fmaf_rn(__fmaf_rn(-q0, scale, d), y, q0);
        // adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and leaves it in the low bits
        const uint32_t code = __float_as_uint(__fadd_rn(fminf(fmaxf(q, 0.0f), 15.0f), 12582912.0f)) & 15;
        packed |= code << (4 * i);
      }
    }
    const int kv = r - a.q_heads, side = value, head = value ? kv - a.pool.kv_heads : kv;
    const int64_t at = a.pool.row(page, side, head) + in_page;
    *reinterpret_cast<uint32_t*>(a.codes + at * (D / 2) + lane * 4) = packed;
    if (lane == 0) a.params[at] = finite ? (__float_as_uint(scale) >> 16) | __float_as_uint(offset) : 0x7fff7fffu;
  }
}

template <int D, typename T, int ROWS>
int launch_rows(const AppendArgs& a, bool vec, bool interleaved, cudaStream_t s) {
  const int64_t per_token = a.q_heads + 2 * (int64_t)a.pool.kv_heads;
  const int64_t groups = a.tokens * ((per_token + ROWS - 1) / ROWS), per_block = kThreads / (D / 8);
  const int64_t blocks = (groups + per_block - 1) / per_block;
  if (blocks > 0x7fffffff) return TANS_E_TOO_LARGE;
  if (vec) {
    if (interleaved) append_kernel<D, T, true, true, ROWS><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    else append_kernel<D, T, true, false, ROWS><<<(unsigned)blocks, kThreads, 0, s>>>(a);
  } else {
    if (interleaved) append_kernel<D, T, false, true, ROWS><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    else append_kernel<D, T, false, false, ROWS><<<(unsigned)blocks, kThreads, 0, s>>>(a);
  }
  note_launch();
  return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
}

// One row for each group of lanes while that does not fill the SMs four times over (a call that waits
// for its memory ends sooner with more of it in flight), else four.
template <int D, typename T>
int launch_append(const AppendArgs& a, bool vec, bool interleaved, cudaStream_t s) {
  const int64_t rows = a.tokens * (a.q_heads + 2 * (int64_t)a.pool.kv_heads);
  const int64_t resident = (int64_t)sm_count() * (2048 / (D / 8));
  return rows <= 4 * resident ? launch_rows<D, T, 1>(a, vec, interleaved, s)
                              : launch_rows<D, T, 4>(a, vec, interleaved, s);
}

// Values of the rows in `slots`: head_dim / 8 lanes for each row.
template <int D, typename T>
__global__ void __launch_bounds__(kThreads) gather_kernel(Pool pool, const int64_t* slots, int64_t tokens, T* k_out,
                                                          T* v_out, uint32_t* status) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x % L;
  const int per_token = 2 * pool.kv_heads;
  const int64_t row = blockIdx.x * (int64_t)(kThreads / L) + threadIdx.x / L;
  if (row >= tokens * per_token) return;
  const int64_t token = row / per_token;
  const int r = (int)(row - token * per_token);
  const int side = r >= pool.kv_heads, head = side ? r - pool.kv_heads : r;
  const int64_t slot = slots[token];
  uint4 w = make_uint4(0, 0, 0, 0);
  if (slot >= pool.num_pages * pool.page_size) {
    if (status && lane == 0) atomicOr(status, TANS_DEV_BAD_INDEX);
  } else if (slot >= 0) {
    const int64_t page = slot / pool.page_size;
    const int64_t at = pool.row(page, side, head) + (slot - page * pool.page_size);
    const uint32_t c = *reinterpret_cast<const uint32_t*>(pool.codes + at * (D / 2) + lane * 4);
    const uint32_t p = pool.params[at];
    const float scale = scale_of(p), offset = offset_of(p);
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = Half2<T>::pack(fmaf((float)((c >> (8 * i)) & 15), scale, offset),
                            fmaf((float)((c >> (8 * i + 4)) & 15), scale, offset));
    }
    w = make_uint4(u[0], u[1], u[2], u[3]);
  }
  *reinterpret_cast<uint4*>((side ? v_out : k_out) + (token * pool.kv_heads + head) * D + lane * 8) = w;
}

// Codes to symbols (and their tables' indexes): 4 codes a thread.
__global__ void __launch_bounds__(kThreads) to_symbols_kernel(Pool pool, const int64_t* page_ids, int64_t n,
                                                              int by_channel, int4* symbols, int4* indexes,
                                                              uint32_t* status) {
  const int64_t row_chunks = (int64_t)pool.page_size * pool.head_dim / 4;
  const int64_t total = n * 2 * pool.kv_heads * row_chunks;
  const int64_t e = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  if (e >= total) return;
  const int64_t row = e / row_chunks, chunk = e - row * row_chunks;
  const int sides = 2 * pool.kv_heads;
  const int64_t i = row / sides;
  const int side = (int)(row - i * sides);
  const int64_t page = page_ids[i];
  uint32_t c = 0;
  if (page < 0 || page >= pool.num_pages) {
    if (status && chunk == 0) atomicOr(status, TANS_DEV_BAD_INDEX);
  } else {
    c = reinterpret_cast<const uint16_t*>(pool.codes)[(page * sides + side) * row_chunks + chunk];
  }
  symbols[e] = make_int4(c & 15, (c >> 4) & 15, (c >> 8) & 15, c >> 12);
  if (indexes) {
    const int t = by_channel ? side * pool.head_dim + (int)(chunk * 4 % pool.head_dim) : side;
    indexes[e] = by_channel ? make_int4(t, t + 1, t + 2, t + 3) : make_int4(t, t, t, t);
  }
}

// Symbols to codes: 8 symbols a thread.
__global__ void __launch_bounds__(kThreads) from_symbols_kernel(const int4* symbols, uint8_t* codes, Pool pool,
                                                                const int64_t* page_ids, int64_t n, uint32_t* status) {
  const int64_t row_chunks = (int64_t)pool.page_size * pool.head_dim / 8;
  const int64_t total = n * 2 * pool.kv_heads * row_chunks;
  const int64_t e = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  if (e >= total) return;
  const int64_t row = e / row_chunks, chunk = e - row * row_chunks;
  const int sides = 2 * pool.kv_heads;
  const int64_t i = row / sides;
  const int side = (int)(row - i * sides);
  const int64_t page = page_ids[i];
  if (page < 0 || page >= pool.num_pages) {
    if (status && chunk == 0) atomicOr(status, TANS_DEV_BAD_INDEX);
    return;
  }
  const int4 a = symbols[2 * e], b = symbols[2 * e + 1];
  if (((a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) & ~15) && status) atomicOr(status, TANS_DEV_BAD_VALUE);
  const uint32_t w = (uint32_t)(a.x & 15) | (a.y & 15) << 4 | (a.z & 15) << 8 | (a.w & 15) << 12 | (b.x & 15) << 16 |
                     (b.y & 15) << 20 | (b.z & 15) << 24 | (uint32_t)(b.w & 15) << 28;
  reinterpret_cast<uint32_t*>(codes)[(page * sides + side) * row_chunks + chunk] = w;
}

bool aligned16(const void* p, int64_t ts, int64_t hs) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
}

}  // namespace
}  // namespace kv4
}  // namespace tans

extern "C" int tans_kv4_append(uint8_t* codes, void* params, int64_t num_pages, int kv_heads, int page_size,
                               int head_dim, int dtype, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                               const void* v, int64_t v_token_stride, int64_t v_head_stride, const void* q,
                               int64_t q_token_stride, int64_t q_head_stride, int q_heads, void* q_out,
                               const int64_t* slots, int64_t tokens, const float* rotation, int64_t rotation_rows,
                               int rotary_dim, const int64_t* positions, int interleaved, uint32_t* dev_status,
                               void* cuda_stream) {
  using namespace tans::kv4;
  if (!pool_ok(codes, params, num_pages, kv_heads, page_size, head_dim) || tokens < 0 ||
      (dtype != TANS_BF16 && dtype != TANS_FP16) || q_heads < 0 || q_heads > 65535)
    return TANS_E_INVALID_ARGUMENT;
  if (!rotation) rotary_dim = 0;
  if (rotation && (rotary_dim < 16 || rotary_dim > head_dim || rotary_dim % 16 != 0 || rotation_rows < 1))
    return TANS_E_INVALID_ARGUMENT;
  if (tokens == 0) return TANS_OK;
  if (!q) q_heads = 0;
  if (!k || !v || !slots || (q && (!q_out || q_heads < 1)) || (rotation && !positions)) return TANS_E_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(rotation)) & 15) != 0)
    return TANS_E_INVALID_ARGUMENT;  // they are read and written 16 bytes at a time
  cudaStream_t s = reinterpret_cast<cudaStream_t>(cuda_stream);
  const AppendArgs a{codes,
                     static_cast<uint32_t*>(params),
                     Pool{codes, static_cast<const uint32_t*>(params), num_pages, kv_heads, page_size, head_dim},
                     q, k, v,
                     q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                     q_out, q_heads, slots, tokens, rotation, rotation_rows, rotary_dim, positions, dev_status};
  const bool vec = aligned16(k, k_token_stride, k_head_stride) && aligned16(v, v_token_stride, v_head_stride) &&
                   (!q || aligned16(q, q_token_stride, q_head_stride));
  const bool il = interleaved != 0;
  if (dtype == TANS_BF16) {
    return head_dim == 64    ? launch_append<64, __nv_bfloat16>(a, vec, il, s)
           : head_dim == 128 ? launch_append<128, __nv_bfloat16>(a, vec, il, s)
                             : launch_append<256, __nv_bfloat16>(a, vec, il, s);
  }
  return head_dim == 64    ? launch_append<64, __half>(a, vec, il, s)
         : head_dim == 128 ? launch_append<128, __half>(a, vec, il, s)
                           : launch_append<256, __half>(a, vec, il, s);
}

extern "C" int tans_kv4_gather(const uint8_t* codes, const void* params, int64_t num_pages, int kv_heads,
                               int page_size, int head_dim, int dtype, const int64_t* slots, int64_t tokens,
                               void* k_out, void* v_out, uint32_t* dev_status, void* cuda_stream) {
  using namespace tans::kv4;
  if (!pool_ok(codes, params, num_pages, kv_heads, page_size, head_dim) || tokens < 0 ||
      (dtype != TANS_BF16 && dtype != TANS_FP16))
    return TANS_E_INVALID_ARGUMENT;
  if (tokens == 0) return TANS_OK;
  if (!slots || !k_out || !v_out || ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15))
    return TANS_E_INVALID_ARGUMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(cuda_stream);
  const Pool pool{codes, static_cast<const uint32_t*>(params), num_pages, kv_heads, page_size, head_dim};
  const int64_t per_block = kThreads / (head_dim / 8);
  const int64_t blocks = (tokens * 2 * kv_heads + per_block - 1) / per_block;
  if (blocks > 0x7fffffff) return TANS_E_TOO_LARGE;
  auto go = [&](auto d, auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    gather_kernel<decltype(d)::value, T><<<(unsigned)blocks, kThreads, 0, s>>>(
        pool, slots, tokens, static_cast<T*>(k_out), static_cast<T*>(v_out), dev_status);
  };
  auto by_dim = [&](auto* t) {
    if (head_dim == 64) go(std::integral_constant<int, 64>{}, t);
    else if (head_dim == 128) go(std::integral_constant<int, 128>{}, t);
    else go(std::integral_constant<int, 256>{}, t);
  };
  if (dtype == TANS_BF16) by_dim(static_cast<__nv_bfloat16*>(nullptr));
  else by_dim(static_cast<__half*>(nullptr));
  tans::note_launch();
  return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
}

extern "C" int tans_kv4_to_symbols(const uint8_t* codes, int64_t num_pages, int kv_heads, int page_size, int head_dim,
                                   const int64_t* page_ids, int64_t n, int by_channel, int32_t* symbols,
                                   int32_t* indexes, uint32_t* dev_status, void* cuda_stream) {
  using namespace tans::kv4;
  if (!pool_ok(codes, codes, num_pages, kv_heads, page_size, head_dim) || n < 0) return TANS_E_INVALID_ARGUMENT;
  if (n == 0) return TANS_OK;
  if (!page_ids || !symbols ||
      ((reinterpret_cast<uintptr_t>(symbols) | reinterpret_cast<uintptr_t>(indexes)) & 15) != 0)
    return TANS_E_INVALID_ARGUMENT;
  const Pool pool{codes, nullptr, num_pages, kv_heads, page_size, head_dim};
  const int64_t threads = n * 2 * kv_heads * ((int64_t)page_size * head_dim / 4);
  const int64_t blocks = (threads + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return TANS_E_TOO_LARGE;
  to_symbols_kernel<<<(unsigned)blocks, kThreads, 0, reinterpret_cast<cudaStream_t>(cuda_stream)>>>(
      pool, page_ids, n, by_channel, reinterpret_cast<int4*>(symbols), reinterpret_cast<int4*>(indexes), dev_status);
  tans::note_launch();
  return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
}

extern "C" int tans_kv4_from_symbols(const int32_t* symbols, uint8_t* codes, int64_t num_pages, int kv_heads,
                                     int page_size, int head_dim, const int64_t* page_ids, int64_t n,
                                     uint32_t* dev_status, void* cuda_stream) {
  using namespace tans::kv4;
  if (!pool_ok(codes, codes, num_pages, kv_heads, page_size, head_dim) || n < 0) return TANS_E_INVALID_ARGUMENT;
  if (n == 0) return TANS_OK;
  if (!page_ids || !symbols || (reinterpret_cast<uintptr_t>(symbols) & 15) != 0) return TANS_E_INVALID_ARGUMENT;
  const Pool pool{codes, nullptr, num_pages, kv_heads, page_size, head_dim};
  const int64_t threads = n * 2 * kv_heads * ((int64_t)page_size * head_dim / 8);
  const int64_t blocks = (threads + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return TANS_E_TOO_LARGE;
  from_symbols_kernel<<<(unsigned)blocks, kThreads, 0, reinterpret_cast<cudaStream_t>(cuda_stream)>>>(
      reinterpret_cast<const int4*>(symbols), codes, pool, page_ids, n, dev_status);
  tans::note_launch();
  return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
}
