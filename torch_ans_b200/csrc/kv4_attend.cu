// kv4_attend.cu -- attention of packed queries over the 4-bit key/value cache: arguments and the
// choice of kernel.
#include <cuda_runtime.h>

#include <algorithm>

#include "kv4_attend.cuh"
#include "launch.cuh"
#include "rans_host.h"

static_assert(tans::kv4::Join::kArrivalBytes == TANS_KV4_ATTEND_COUNTS, "the header names the size");

namespace {
// Whether the kernel that is bound by the cache's bytes takes the call: `rows` query rows at most share a
// key/value head.  It reads the cache once for each 8 or 16 of them, the other unpacks it once for 128 or
// 256.  Measured for head_dim 64, 128, 256: 16 contexts of 8,192 tokens with 4 heads, 32 rows 52, 62 and
// 113 us against 78, 88 and 212, 48 rows 70, 81 and 158 against 109, 125 and 213, 64 rows 83, 103 and 205
// against 109, 125 and 213, 96 rows 115, 145 and 297 against 109, 127 and 270; 64 contexts of 700 tokens with 8
// heads, 32 rows 45, 68 and 115 us against 63, 76 and 124, 48 rows 63, 88 and 167 against 64, 78 and 126, 64
// rows 80, 110 and 212 against 64, 78 and 127.  Long contexts would take this kernel up to 64 rows and short ones up
// to 32: the rule looks at the rows alone.
bool few_rows(int64_t rows) { return rows <= 48; }
}  // namespace

extern "C" size_t tans_kv4_attend_workspace_size(int64_t total_queries, int q_heads, int kv_heads, int head_dim,
                                                 int64_t batch, int64_t max_pages, int page_size, int64_t max_queries) {
  using namespace tans::kv4;
  if (total_queries < 1 || kv_heads < 1 || q_heads < kv_heads) return 0;
  const int64_t rows = std::min(max_queries, total_queries) * (q_heads / kv_heads);
  return few_rows(rows) ? attend_rows_workspace(head_dim, rows)
                        : attend_prompt_workspace(head_dim, total_queries * (q_heads / kv_heads),
                                                  std::min(batch, total_queries), kv_heads, max_pages * page_size);
}

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
  if (!q || !out || (batch > 0 && (!lengths || (max_pages > 0 && !pages))) || (!q_starts && batch != total_queries) ||
      ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0)
    return TANS_E_INVALID_ARGUMENT;
  // token and query numbers are 32-bit in the kernels, with room for a tile past the end
  if (total_queries > (1 << 30) / q_heads || batch > (1 << 30) || max_pages > (1 << 30) / page_size ||
      num_pages > 0x7fffffff)
    return TANS_E_TOO_LARGE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(cuda_stream);
  const int group = q_heads / kv_heads;
  const bool vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
  const AttendArgs a{Pool{codes, static_cast<const uint32_t*>(params), num_pages, kv_heads, page_size, head_dim},
                     q, q_token_stride, q_head_stride, total_queries, q_heads,
                     Divider::of(group), Divider::of(kv_heads), Divider::of(page_size), pages, batch, max_pages, lengths,
                     q_starts, scale * 1.4426950408889634f, causal, vec, out, lse, dev_status,
                     std::min(tans::env_int("TORCH_ANS_B200_WAIT_LIMIT", 1 << 20), 1 << 30)};
  const int64_t most = std::min(max_queries, total_queries);
  const size_t need = tans_kv4_attend_workspace_size(total_queries, q_heads, kv_heads, head_dim, batch, max_pages,
                                                     page_size, max_queries);
  void* ws = workspace;
  if (!ws) {
    if (cudaMallocAsync(&ws, need, s) != cudaSuccess) return TANS_E_CUDA;
    if (cudaMemsetAsync(ws, 0, Join::kArrivalBytes, s) != cudaSuccess) {
      cudaFreeAsync(ws, s);
      return TANS_E_CUDA;
    }
  } else if (workspace_bytes < need) {
    return TANS_E_WORKSPACE;
  }
  const int rc = few_rows(most * group) ? launch_attend_rows(a, dtype, most * group, ws, s)
                                        : launch_attend_prompt(a, dtype, ws, s);
  if (!workspace) cudaFreeAsync(ws, s);
  return rc;
}
