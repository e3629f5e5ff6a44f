// kv4_attend.cuh -- what the attention kernels over the 4-bit cache share.
#pragma once

#include <cuda_runtime.h>

#include "kv4.cuh"

namespace tans {
namespace kv4 {

struct AttendArgs {
  Pool pool;
  const void* q;
  int64_t q_ts, q_hs;  // strides of a token and a head, in elements
  int64_t total_queries;
  int q_heads;
  Divider group, kv_heads, page_size;  // query heads that share a key/value head; the pool's
  const int32_t* pages;
  int64_t batch, max_pages;
  const int32_t* lengths;
  const int32_t* q_starts;
  float scale_log2;  // the score's factor times log2(e): softmax is taken in powers of two
  int causal;
  int vec;  // rows of q start on 16 bytes
  void* out;
  float* lse;
  uint32_t* status;
  int wait_limit;  // tries of a wait of one warp for another, a microsecond each at most
};

// One sequence: its tokens, its queries (first and number); not ok: its starts are out of order or past the
// queries, and it has none.
struct Sequence {
  int length, start, count;
  bool ok;
};

__device__ __forceinline__ void flag(uint32_t* status, uint32_t bit) {
  if (status) atomicOr(status, bit);
}

__device__ __forceinline__ Sequence sequence(const AttendArgs& a, int64_t b, bool report) {
  Sequence s;
  s.ok = true;
  if (a.q_starts) {
    const int lo = a.q_starts[b], hi = a.q_starts[b + 1];
    s.ok = lo >= 0 && hi >= lo && hi <= a.total_queries;
    if (!s.ok && report) flag(a.status, TANS_DEV_BAD_VALUE);
    s.start = s.ok ? lo : 0;
    s.count = s.ok ? hi - lo : 0;
  } else {
    s.start = (int)b;
    s.count = 1;
  }
  const int length = a.lengths[b];
  const int64_t most = a.max_pages * a.pool.page_size;
  s.length = length < 0 ? 0 : (length > most ? (int)most : length);
  if (s.length != length && report) flag(a.status, TANS_DEV_BAD_VALUE);
  return s;
}

// Queries before the first start and after the last belong to no sequence: zeros, shared by all
// threads of the grid.
template <typename T>
__device__ __forceinline__ void zero_unowned(const AttendArgs& a, int dim, int64_t thread, int64_t threads) {
  if (!a.q_starts) return;
  const int64_t first = max(0, min((int)a.total_queries, a.q_starts[0]));
  const int64_t last = max((int)first, min((int)a.total_queries, a.q_starts[a.batch]));
  const int64_t heads = a.q_heads, unowned = (first + a.total_queries - last) * heads;
  if (unowned == 0) return;
  for (int64_t e = thread; e < unowned * dim; e += threads) {
    const int64_t row = e / dim, at = row < first * heads ? row : row + (last - first) * heads;
    static_cast<T*>(a.out)[at * dim + e % dim] = Half2<T>::round(0.0f);
    if (a.lse && e % dim == 0) a.lse[at] = -INFINITY;
  }
}

// For starts that are not in order: queries that no sequence answers, one at a time by some threads, become
// zeros.  `tiles` row tiles of `rows` rows are answered, in the order of the sequences.
static __device__ __noinline__ void zero_unanswered(const int32_t* q_starts, int64_t batch, int64_t total_queries, int group,
                                                    int64_t row_elements, uint16_t* out, float* lse, int q_heads,
                                                    int64_t thread, int64_t threads, int rows, int64_t tiles) {
  for (int64_t i = thread; i < total_queries; i += threads) {
    bool answered = false;
    int64_t before = 0;
    for (int64_t b = 0; b < batch && !answered; ++b) {
      const int lo = q_starts ? q_starts[b] : (int)b, hi = q_starts ? q_starts[b + 1] : (int)b + 1;
      if (lo < 0 || hi < lo || hi > total_queries) continue;
      before += ((int64_t)(hi - lo) * group + rows - 1) / rows;
      answered = i >= lo && i < hi && before <= tiles;
    }
    if (answered) continue;
    for (int64_t e = 0; e < row_elements; ++e) out[i * row_elements + e] = 0;
    for (int h = 0; lse && h < q_heads; ++h) lse[i * q_heads + h] = -INFINITY;
  }
}
__device__ __forceinline__ void zero_unanswered(const AttendArgs& a, int dim, int64_t thread, int64_t threads, int rows,
                                                int64_t tiles) {
  zero_unanswered(a.q_starts, a.batch, a.total_queries, a.group.d, (int64_t)a.q_heads * dim, static_cast<uint16_t*>(a.out),
                  a.lse, a.q_heads, thread, threads, rows, tiles);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 2^x for a whole number x in -126 .. 127
__device__ __forceinline__ float pow2(int x) { return __int_as_float((x + 127) << 23); }

// Where the parts of a row tile that several blocks share are joined.  Blocks take equal, contiguous
// shares of all (sequence, row tile, head, token) work, so a tile's blocks are neighbours c0 .. c1.
// Each leaves its sums in one of its two places (1: the tile starts in this block, 0: it started
// before), and the last of them to arrive joins them, in the order of the blocks whatever the order
// of arrival, so results repeat.  Over kFan blocks join in two levels.  The counts of arrivals are
// zero between launches: the last arrival takes its count back.
constexpr int kFan = 16;
constexpr int kMostBlocks = 4 * 160;  // blocks that a workspace has places for

struct Join {
  int* arrivals;  // [2 levels][kMostBlocks][2]
  float2* stats;  // [kMostBlocks][2][rows]: maximum (a power of two's exponent) and sum
  float* parts;   // [kMostBlocks][2][rows][dim]

  static size_t bytes(int64_t rows, int64_t dim) {
    return kArrivalBytes + (size_t)kMostBlocks * 2 * rows * (8 + dim * 4);
  }
  static constexpr size_t kArrivalBytes = 2 * kMostBlocks * 2 * sizeof(int);
  static Join in(void* workspace, int64_t rows) {
    Join j;
    j.arrivals = static_cast<int*>(workspace);
    j.stats = reinterpret_cast<float2*>(static_cast<char*>(workspace) + kArrivalBytes);
    j.parts = reinterpret_cast<float*>(j.stats + kMostBlocks * 2 * rows);
    return j;
  }
};

__device__ __forceinline__ bool arrive(int* count, int expected) {
  if (atomicAdd(count, 1) + 1 < expected) return false;
  *count = 0;  // nobody else comes in this launch
  return true;
}

int launch_attend_rows(const AttendArgs& a, int dtype, int64_t max_rows, void* workspace, cudaStream_t s);
size_t attend_rows_workspace(int head_dim, int64_t max_rows);
int launch_attend_prompt(const AttendArgs& a, int dtype, void* workspace, cudaStream_t s);
size_t attend_prompt_workspace(int head_dim, int64_t total_rows, int64_t batch, int kv_heads, int64_t max_tokens);

}  // namespace kv4
}  // namespace tans
