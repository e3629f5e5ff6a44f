// kv4_attend.cu -- attention of packed queries over the 4-bit key/value cache.
#include <cuda_runtime.h>

#include "kv4.cuh"
#include "launch.cuh"
#include "rans_host.h"

namespace tans {
namespace kv4 {
namespace {

struct AttendArgs {
  Pool pool;
  const void* q;
  int64_t q_ts, q_hs;
  int64_t total_queries;
  int q_heads;
  const int32_t* pages;
  int64_t batch, max_pages;
  const int32_t* lengths;
  const int32_t* q_starts;
  float scale;
  int causal;
  void* out;
  float* lse;
  uint32_t* status;
};

__device__ __forceinline__ void flag(uint32_t* status, uint32_t bit) {
  if (status) atomicOr(status, bit);
}

// One block for each query and head: four warps share the tokens, each with its own running maximum
// and sum; a lane holds head_dim / 32 channels.
template <int D, typename T>
__global__ void __launch_bounds__(128) attend_kernel(AttendArgs a) {
  constexpr int C = D / 32;
  const int64_t i = blockIdx.x;
  const int h = blockIdx.y, kvh = h / (a.q_heads / a.pool.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float sh_m[4], sh_l[4], sh_o[4][D];

  int64_t b = -1, start = 0, count = 1;
  if (a.q_starts) {
    for (int64_t j = 0; j < a.batch; ++j) {
      const int32_t lo = a.q_starts[j], hi = a.q_starts[j + 1];
      if (lo < 0 || hi < lo || hi > a.total_queries) {
        if (threadIdx.x == 0) flag(a.status, TANS_DEV_BAD_VALUE);
      } else if (i >= lo && i < hi) {
        b = j;
        start = lo;
        count = hi - lo;
        break;
      }
    }
  } else {
    b = i;
    start = i;
  }
  int64_t length = b >= 0 ? a.lengths[b] : 0;
  const int64_t most = a.max_pages * a.pool.page_size;
  if (length < 0 || length > most) {
    if (threadIdx.x == 0) flag(a.status, TANS_DEV_BAD_VALUE);
    length = length < 0 ? 0 : most;
  }
  const int64_t end = a.causal ? min(length, length - count + (i - start) + 1) : length;

  float q[C], o[C];
  const T* qp = static_cast<const T*>(a.q) + i * a.q_ts + h * a.q_hs + lane * C;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    q[c] = Half2<T>::load(qp + c);
    o[c] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t t = warp; t < end; t += 4) {
    const int64_t page = a.pages[b * a.max_pages + t / a.pool.page_size];
    if (page < 0 || page >= a.pool.num_pages) {
      if (lane == 0) flag(a.status, TANS_DEV_BAD_INDEX);
      continue;
    }
    const int64_t kr = a.pool.row(page, 0, kvh) + t % a.pool.page_size;
    const int64_t vr = a.pool.row(page, 1, kvh) + t % a.pool.page_size;
    const uint32_t kp = a.pool.params[kr], vp = a.pool.params[vr];
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      const uint32_t w = a.pool.codes[kr * (D / 2) + (lane * C + c) / 2];
      s = fmaf(q[c], fmaf((float)(w & 15), scale_of(kp), offset_of(kp)), s);
      s = fmaf(q[c + 1], fmaf((float)(w >> 4), scale_of(kp), offset_of(kp)), s);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.scale;
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.0f : expf(m - top), p = expf(s - top);
    l = l * keep + p;
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      const uint32_t w = a.pool.codes[vr * (D / 2) + (lane * C + c) / 2];
      o[c] = fmaf(p, fmaf((float)(w & 15), scale_of(vp), offset_of(vp)), o[c] * keep);
      o[c + 1] = fmaf(p, fmaf((float)(w >> 4), scale_of(vp), offset_of(vp)), o[c + 1] * keep);
    }
    m = top;
  }
  if (lane == 0) {
    sh_m[warp] = m;
    sh_l[warp] = l;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) sh_o[warp][lane * C + c] = o[c];
  __syncthreads();
  const float top = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
  float w[4], sum = 0.0f;
  for (int j = 0; j < 4; ++j) {
    w[j] = sh_m[j] == -INFINITY ? 0.0f : expf(sh_m[j] - top);
    sum += w[j] * sh_l[j];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float v = 0.0f;
    for (int j = 0; j < 4; ++j)
      if (w[j] > 0.0f) v += w[j] * sh_o[j][d];
    static_cast<T*>(a.out)[(i * a.q_heads + h) * D + d] = Half2<T>::round(sum != 0.0f ? v / sum : 0.0f);
  }
  if (threadIdx.x == 0 && a.lse) a.lse[i * a.q_heads + h] = sum != 0.0f ? top + logf(sum) : -INFINITY;
}

}  // namespace
}  // namespace kv4
}  // namespace tans

extern "C" size_t tans_kv4_attend_workspace_size(int64_t, int, int, int, int64_t, int64_t, int, int64_t) { return 0; }

extern "C" int tans_kv4_attend(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t total_queries,
                               int q_heads, int dtype, const uint8_t* codes, const void* params, int64_t num_pages,
                               int kv_heads, int page_size, int head_dim, const int32_t* pages, int64_t batch,
                               int64_t max_pages, const int32_t* lengths, const int32_t* q_starts, int64_t max_queries,
                               float scale, int causal, void* out, float* lse, void* workspace,
                               size_t workspace_bytes, uint32_t* dev_status, void* cuda_stream) {
  using namespace tans::kv4;
  if (!pool_ok(codes, params, num_pages, kv_heads, page_size, head_dim) || total_queries < 0 || batch < 0 ||
      max_pages < 0 || (dtype != TANS_BF16 && dtype != TANS_FP16) || q_heads < 1 || q_heads > 65535 ||
      q_heads % kv_heads != 0 || max_queries < 0)
    return TANS_E_INVALID_ARGUMENT;
  if (total_queries == 0) return TANS_OK;
  if (!q || !out || (batch > 0 && (!lengths || (max_pages > 0 && !pages))) || (!q_starts && batch != total_queries))
    return TANS_E_INVALID_ARGUMENT;
  const AttendArgs a{Pool{codes, static_cast<const uint32_t*>(params), num_pages, kv_heads, page_size, head_dim},
                     q, q_token_stride, q_head_stride, total_queries, q_heads, pages, batch, max_pages, lengths,
                     q_starts, scale, causal, out, lse, dev_status};
  if (total_queries > 0x7fffffff) return TANS_E_TOO_LARGE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(cuda_stream);
  const dim3 grid((unsigned)total_queries, (unsigned)q_heads);
  auto by_dim = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (head_dim == 64) attend_kernel<64, T><<<grid, 128, 0, s>>>(a);
    else if (head_dim == 128) attend_kernel<128, T><<<grid, 128, 0, s>>>(a);
    else attend_kernel<256, T><<<grid, 128, 0, s>>>(a);
  };
  if (dtype == TANS_BF16) by_dim(static_cast<__nv_bfloat16*>(nullptr));
  else by_dim(static_cast<__half*>(nullptr));
  tans::note_launch();
  return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
}
