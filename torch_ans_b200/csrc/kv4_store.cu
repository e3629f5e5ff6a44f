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

// A slot's page.  Pools of 2^31 slots or more take the long division.
struct PageOf {
  Divider divider;
  bool small;
  int page_size;
  static PageOf of(const Pool& p) {
    return {Divider::of((uint32_t)p.page_size), p.num_pages < ((int64_t)1 << 31) / p.page_size, p.page_size};
  }
  __device__ __forceinline__ int64_t operator()(int64_t slot) const {
    return small ? (int64_t)divider.div((int)slot) : slot / page_size;
  }
};

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
  PageOf page_of;
  Divider chunks;  // groups of rows of a token
};

// 4 consecutive elements of a row, as they are, and as floats
template <typename T, bool VEC>
__device__ __forceinline__ uint2 load4(const T* p) {
  if constexpr (VEC) return *reinterpret_cast<const uint2*>(p);
  const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
  return make_uint2(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16);
}
template <typename T>
__device__ __forceinline__ void floats(const uint2& w, float2 (&x)[2]) {
  x[0] = Half2<T>::unpack(w.x);
  x[1] = Half2<T>::unpack(w.y);
}

// (a, b) turned by an angle, every product and sum rounded by itself
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
}

// Rotation and quantisation, head_dim / 8 lanes for each row (one token's head), 8 channels a lane in two
// fours: channels that turn together are in one lane (i and i + rotary / 2, or neighbours), so nothing is
// exchanged for the rotation.  A group of lanes takes ROWS rows of one token, so that the token's cosines
// and sines are read once for all of them and the loads of the rows do not wait for one another.
//
// What it may not do without is bytes: 2 read and 2 written for a query's channel, 2 read and about 0.53
// written for a key's or a value's.  16,381 tokens of 32 + 16 heads of 128 (355 MB) take 95 us, 3.7 TB/s:
// warps wait for their loads (the largest stall) and for one another's turn, with 0.69 instructions a
// scheduler and cycle (about 160 for two rows of a warp).  With 2 rows a group 112 us, with 8 about 140 (too
// few groups at once).  The products and sums of the rotation are rounded one by one (no
// fused multiply-add), so the codes do not depend on the compiler's choices.
//
// The quotient (x - offset) / scale is the correctly rounded one, so that ties (common: x has 8 or 11
// bits, scale 8) go to the even code; it takes one division a row and, by Markstein's theorem, two fused
// steps a channel: with y the correctly rounded 1 / scale and q0 = d y, q0 + (d - q0 scale) y rounds
// correctly.
template <int D, typename T, bool VEC, bool INTERLEAVED, int ROWS>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x % L, half = a.rotary / 2;
  const bool in_rotary = lane * 8 < a.rotary;
  const int d0 = !INTERLEAVED && in_rotary ? lane * 4 : lane * 8, d1 = !INTERLEAVED && in_rotary ? d0 + half : d0 + 4;
  const int per_token = a.q_heads + 2 * a.pool.kv_heads;
  const int group = blockIdx.x * (kThreads / L) + threadIdx.x / L, of = a.chunks.div(group);
  const int64_t token = min((int64_t)of, a.tokens - 1);  // groups past the end keep the warp's shuffles whole
  const int r0 = (group - of * (int)a.chunks.d) * ROWS;
  const int rows = of >= a.tokens ? 0 : min(ROWS, per_token - r0);

  const T* q_at = static_cast<const T*>(a.q) + token * a.q_ts;
  const T* k_at = static_cast<const T*>(a.k) + token * a.k_ts - a.q_heads * a.k_hs;
  const T* v_at = static_cast<const T*>(a.v) + token * a.v_ts - (a.q_heads + a.pool.kv_heads) * a.v_hs;
  uint2 raw0[ROWS], raw1[ROWS];
#pragma unroll
  for (int n = 0; n < ROWS; ++n) {  // rows of the token: queries, keys, values
    const int r = r0 + n;
    raw0[n] = raw1[n] = make_uint2(0, 0);
    if (n < rows) {
      const T* src = r < a.q_heads ? q_at + r * a.q_hs : (r < a.q_heads + a.pool.kv_heads ? k_at + r * a.k_hs : v_at + r * a.v_hs);
      raw0[n] = load4<T, VEC>(src + d0);
      raw1[n] = load4<T, VEC>(src + d1);
    }
  }

  const int64_t slot = r0 + rows > a.q_heads ? a.slots[token] : -1;
  bool turns = false;
  float2 c[2], s[2];  // of the lane's four angles
  if (a.rotary > 0) {
    const int64_t pos = a.positions[token];
    const bool known = pos >= 0 && pos < a.rotation_rows;
    if (!known && a.status && lane == 0 && r0 == 0 && rows > 0) atomicOr(a.status, TANS_DEV_BAD_INDEX);
    turns = known && in_rotary;
    if (turns) {
      const float* cosines = a.rotation + pos * a.rotary + lane * 4;
      const float4 x = *reinterpret_cast<const float4*>(cosines), y = *reinterpret_cast<const float4*>(cosines + half);
      c[0] = make_float2(x.x, x.y);
      c[1] = make_float2(x.z, x.w);
      s[0] = make_float2(y.x, y.y);
      s[1] = make_float2(y.z, y.w);
    }
  }
  bool stores = slot >= 0;
  if (slot >= a.pool.num_pages * a.pool.page_size) {
    stores = false;
    if (a.status && lane == 0) atomicOr(a.status, TANS_DEV_BAD_INDEX);
  }
  const int64_t page = stores ? a.page_of(slot) : 0;
  const int in_page = stores ? (int)(slot - page * a.pool.page_size) : 0;

#pragma unroll
  for (int n = 0; n < ROWS; ++n) {
    const int r = r0 + n;
    const bool live = n < rows, query = r < a.q_heads, value = r >= a.q_heads + a.pool.kv_heads;
    float2 u[2], w[2];  // the lane's fours
    floats<T>(raw0[n], u);
    floats<T>(raw1[n], w);
    if (turns && !value) {
      if constexpr (INTERLEAVED) {
        turn(u[0].x, u[0].y, c[0].x, s[0].x);
        turn(u[1].x, u[1].y, c[0].y, s[0].y);
        turn(w[0].x, w[0].y, c[1].x, s[1].x);
        turn(w[1].x, w[1].y, c[1].y, s[1].y);
      } else {
        turn(u[0].x, w[0].x, c[0].x, s[0].x);
        turn(u[0].y, w[0].y, c[0].y, s[0].y);
        turn(u[1].x, w[1].x, c[1].x, s[1].x);
        turn(u[1].y, w[1].y, c[1].y, s[1].y);
      }
    }
    if (query && live) {
      T* dst = static_cast<T*>(a.q_out) + (token * a.q_heads + r) * D;
      *reinterpret_cast<uint2*>(dst + d0) = make_uint2(Half2<T>::pack(u[0].x, u[0].y), Half2<T>::pack(u[1].x, u[1].y));
      *reinterpret_cast<uint2*>(dst + d1) = make_uint2(Half2<T>::pack(w[0].x, w[0].y), Half2<T>::pack(w[1].x, w[1].y));
    }
    if (__all_sync(0xffffffffu, query || !live || !stores)) continue;
    const float x[8] = {u[0].x, u[0].y, u[1].x, u[1].y, w[0].x, w[0].y, w[1].x, w[1].y};

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
    // The format's scale is this product, not a quotient: they differ by a unit in float's last place, which
    // decides where a quotient would lie half way between two bfloat16 numbers (0.06 % of random float16 rows).
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
    *reinterpret_cast<uint16_t*>(a.codes + at * (D / 2) + d0 / 2) = (uint16_t)packed;
    *reinterpret_cast<uint16_t*>(a.codes + at * (D / 2) + d1 / 2) = (uint16_t)(packed >> 16);
    if (lane == 0) a.params[at] = finite ? (__float_as_uint(scale) >> 16) | __float_as_uint(offset) : 0x7fff7fffu;
  }
}

template <int D, typename T, int ROWS>
int launch_rows(AppendArgs a, bool vec, bool interleaved, cudaStream_t s) {
  const int64_t chunks = (a.q_heads + 2 * (int64_t)a.pool.kv_heads + ROWS - 1) / ROWS, per_block = kThreads / (D / 8);
  const int64_t blocks = (a.tokens * chunks + per_block - 1) / per_block;
  if (blocks > 0x7fffffff / per_block) return TANS_E_TOO_LARGE;  // groups are numbered in 31 bits
  a.chunks = Divider::of((uint32_t)chunks);
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

// Values of the rows in `slots`: head_dim / 8 lanes for each row.  16,381 tokens of 16 rows of 128 (85 MB,
// four fifths of them written) take 26 us, 3.2 TB/s: a lane's slot, codes and parameters are three loads in a row
// with nothing else in flight (they are by far the largest stall).
template <int D, typename T>
__global__ void __launch_bounds__(kThreads) gather_kernel(Pool pool, PageOf page_of, Divider per_token,
                                                          const int64_t* slots, int64_t tokens, T* k_out, T* v_out,
                                                          uint32_t* status) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x % L;
  const int row = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int token = per_token.div(row);
  if (token >= tokens) return;
  const int r = row - token * (int)per_token.d;
  const int side = r >= pool.kv_heads, head = side ? r - pool.kv_heads : r;
  const int64_t slot = slots[token];
  uint4 w = make_uint4(0, 0, 0, 0);
  if (slot >= pool.num_pages * pool.page_size) {
    if (status && lane == 0) atomicOr(status, TANS_DEV_BAD_INDEX);
  } else if (slot >= 0) {
    const int64_t page = page_of(slot);
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
  *reinterpret_cast<uint4*>((side ? v_out : k_out) + ((int64_t)token * pool.kv_heads + head) * D + lane * 8) = w;
}

// Codes to symbols (and their tables' indexes): 4 codes a thread, 16 bytes of each output at a time.  A row
// of a page has a multiple of 1,024 codes (16 tokens of 64 channels at least), so a block's 256 threads are
// in one row and only the block finds out where.  Bound by the 8 bytes written for each code: 67 million
// codes in 100 us, 5.7 TB/s (111 us when each thread found its row).
__global__ void __launch_bounds__(kThreads) to_symbols_kernel(Pool pool, const int64_t* page_ids, int by_channel,
                                                              int4* symbols, int4* indexes, uint32_t* status) {
  const unsigned row_blocks = (unsigned)(pool.page_size * (pool.head_dim / 4) / kThreads);
  const unsigned row = blockIdx.x / row_blocks, sides = 2 * pool.kv_heads, i = row / sides, side = row - i * sides;
  const unsigned chunk = (blockIdx.x - row * row_blocks) * kThreads + threadIdx.x;
  const int64_t page = page_ids[i], e = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  uint32_t c = 0;
  if (page < 0 || page >= pool.num_pages) {
    if (status && chunk == 0) atomicOr(status, TANS_DEV_BAD_INDEX);
  } else {
    c = reinterpret_cast<const uint16_t*>(pool.codes)[(page * sides + side) * (row_blocks * (int64_t)kThreads) + chunk];
  }
  __stcs(symbols + e, make_int4(c & 15, (c >> 4) & 15, (c >> 8) & 15, c >> 12));
  if (indexes) {
    const int t = by_channel ? side * pool.head_dim + (chunk * 4 & (pool.head_dim - 1)) : side;
    __stcs(indexes + e, by_channel ? make_int4(t, t + 1, t + 2, t + 3) : make_int4(t, t, t, t));
  }
}

// Symbols to codes: 8 symbols a thread, a block in one row as above.  Bound by the 4 bytes read for each: 67
// million in 42 to 47 us, 6.4 TB/s.
constexpr int kBackThreads = 128;
__global__ void __launch_bounds__(kBackThreads) from_symbols_kernel(const int4* symbols, uint8_t* codes, Pool pool,
                                                                    const int64_t* page_ids, uint32_t* status) {
  const unsigned row_blocks = (unsigned)(pool.page_size * (pool.head_dim / 8) / kBackThreads);
  const unsigned row = blockIdx.x / row_blocks, sides = 2 * pool.kv_heads, i = row / sides, side = row - i * sides;
  const unsigned chunk = (blockIdx.x - row * row_blocks) * kBackThreads + threadIdx.x;
  const int64_t page = page_ids[i], e = blockIdx.x * (int64_t)kBackThreads + threadIdx.x;
  const int4 a = __ldcs(symbols + 2 * e), b = __ldcs(symbols + 2 * e + 1);
  if (page < 0 || page >= pool.num_pages) {
    if (status && chunk == 0) atomicOr(status, TANS_DEV_BAD_INDEX);
    return;
  }
  if (((a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) & ~15) && status) atomicOr(status, TANS_DEV_BAD_VALUE);
  const uint32_t w = (uint32_t)(a.x & 15) | (a.y & 15) << 4 | (a.z & 15) << 8 | (a.w & 15) << 12 | (b.x & 15) << 16 |
                     (b.y & 15) << 20 | (b.z & 15) << 24 | (uint32_t)(b.w & 15) << 28;
  reinterpret_cast<uint32_t*>(codes)[(page * sides + side) * (row_blocks * (int64_t)kBackThreads) + chunk] = w;
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
  AppendArgs a{codes,
                     static_cast<uint32_t*>(params),
                     Pool{codes, static_cast<const uint32_t*>(params), num_pages, kv_heads, page_size, head_dim},
                     q, k, v,
                     q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                     q_out, q_heads, slots, tokens, rotation, rotation_rows, rotary_dim, positions, dev_status, {}, {}};
  a.page_of = PageOf::of(a.pool);
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
  if (blocks > 0x7fffffff / per_block) return TANS_E_TOO_LARGE;  // rows are numbered in 31 bits
  auto go = [&](auto d, auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    gather_kernel<decltype(d)::value, T><<<(unsigned)blocks, kThreads, 0, s>>>(
        pool, PageOf::of(pool), Divider::of(2u * kv_heads), slots, tokens, static_cast<T*>(k_out), static_cast<T*>(v_out), dev_status);
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
      pool, page_ids, by_channel, reinterpret_cast<int4*>(symbols), reinterpret_cast<int4*>(indexes), dev_status);
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
  const int64_t blocks = threads / kBackThreads;
  if (blocks > 0x7fffffff) return TANS_E_TOO_LARGE;
  from_symbols_kernel<<<(unsigned)blocks, kBackThreads, 0, reinterpret_cast<cudaStream_t>(cuda_stream)>>>(
      reinterpret_cast<const int4*>(symbols), codes, pool, page_ids, dev_status);
  tans::note_launch();
  return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
}
