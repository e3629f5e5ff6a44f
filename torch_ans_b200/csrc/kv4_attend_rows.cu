// kv4_attend_rows.cu -- attention over the 4-bit cache when few queries share a key/value head (one
// token of a sequence, or a few drafted ones): bound by the bytes of the cache, so the work is split
// over the tokens and a code costs as few instructions as the tensor cores' operands allow.
//
// A warp takes 32 tokens at a time for up to 8 (or 16) query rows of one key/value head.  Both
// products are mma.sync.m16n8k16 with the cache as the 16-row operand, so 8 columns of rows cost no
// more than one: S^T = K Q^T (16 tokens x 16 channels) and O^T = V^T P^T (16 channels x 16 tokens).
// Codes become float16 by masking alone: the bits of c in the low four bits of a half are the
// subnormal c * 2^-24, in the next four c * 2^-20; the tensor cores take subnormals exactly, and the
// powers of two go into the queries (keys) and the result (values).  That is 5 instructions for 8
// codes of a key word (four masks, one shift), and 12 for 16 codes of two tokens' value words (two
// byte permutes pair the tokens of a channel first).
//
// With a row's (s, o): q.k = s (q.c) + o sum(q), so scales and offsets never touch the codes: the
// score x (a power of two's exponent) takes two products and one sum, and the value's scale goes into
// the weight,
//   sum 2^x v = 2^Y (sum w c - 7.5 sum w) + sum 2^x (o + 7.5 s),  w = float16(2^(x - Y) s).
// The 7.5 centres the codes (sum w is one more row of ones in the second product), so a weight's
// rounding to float16 (2^-11) weighs on the code's distance from the middle, not on the code: about half
// the error.  The sums of the softmax, the offsets and all accumulators are float.  A query row is
// brought under 2^14 by a power of two and rounded to float16, which loses nothing that bfloat16 or
// float16 holds above 2^-24 of the row's largest.
//
// Y is each query row's own.  It follows the largest product of a weight and a value's size, max(s, |o +
// 7.5 s|), among the tokens that the row sees, and leaves it at most 2^6 when it moves: what float16 cuts
// off is 2^-31 of the largest product, whatever the sizes of the values and of those that do not count
// (hidden tokens, or ones of no weight).  Weights 2^(x - R) are taken against R = Y, or the running
// maximum m of x where that is less: then they are at most 2^8 and w = 2^(x - R) (s 2^(R - Y)); Y is kept
// above m - 96, so where values are tiny the weights stay in float's range.  m and Y move only when a score
// passes m by over 8, or when a lane's largest score and largest size (of four tokens) together pass Y by
// 14 (w is then under 2^15): most steps compare and go on.  Where |m| passes 2^10 the column's scores get an
// origin, their largest one itself, taken off before anything else is added to them: equal scores stay equal, in
// whatever warp, and Y and R as exact as they are.
//
// Measured: 48 contexts of 256 to 16,384 tokens (222k together, 32 query and 8 key/value heads of 128, 242
// MB) 75 us, 3.2 TB/s: about 570 instructions a step, the ALU pipe half busy, and each item's start and end;
// 3 contexts of about 127k tokens (16 and 2 heads, 103 MB) 43 us, of which the steps are about 20 (5 to 6
// TB/s), the start 6 and the joins of 97 blocks an item 10; one context of 777 tokens 12 us, all latency.
// With one factor for all rows of a warp instead of a Y for each row the ragged batch took 72 us, and a value 2^20
// times larger than the others, of no weight or hidden, took a fifth of the answers away.
// Blocks of 4 warps, four on an SM, so that one's start and end run beside the others' steps: with 8 warps,
// two on an SM, the ragged batch took 83 us and the long contexts 44 when these took 72 and 43.
#include "kv4_attend.cuh"
#include "launch.cuh"
#include "rans_host.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace tans {
namespace kv4 {
namespace {

constexpr int kWarps = 4;
constexpr int kStep = 32;   // tokens a warp takes at a time
constexpr int kStages = 3;  // steps in flight for each warp, the one in use among them
constexpr float kSlack = 8.0f;     // by which a score may pass the running maximum
constexpr float kRoom = 14.0f;     // by which a product's size may pass Y: its weight is under 2^15
constexpr float kDeepest = 96.0f;  // Y is at most so far under m: weights and their sums stay in float's range
constexpr float kHighest = 122.0f; // and at most so far above it: a size of 2^128 at a weight of 2^8 leaves 2^14
constexpr float kNone = -1e30f;    // Y before the first token
constexpr float kFar = 1024.0f;    // |m| from which on scores have an origin
constexpr int kItemSteps = 8;  // what an item's start and end cost a block, in steps
constexpr int kMostParts = kMostBlocks / kFan > kFan ? kMostBlocks / kFan : kFan;  // that are joined at a time

// A step of a warp in shared memory: 32 key rows, 32 value rows, 32 + 32 parameters.
template <int D>
struct Stage {
  static constexpr int ROW = D / 2, CHUNKS = D / 32;  // bytes, 16-byte chunks of a row
  static constexpr int COPIES = CHUNKS / 2;           // chunks of 16 rows for each lane
  static constexpr int K = 0, V = kStep * ROW, KP = 2 * kStep * ROW, VP = KP + kStep * 4, BYTES = VP + kStep * 4;

  // Where a 16-byte chunk of a token's row lies.  Key rows are read by lane 4 g + t as the t-th
  // quarter of row token(g), value rows as the g-th eighth of rows t + 4 j; the order of rows and
  // chunks puts the lanes of one access on different banks for both.
  static __device__ __forceinline__ int place(int token, int chunk) {
    if constexpr (D == 64) return (token ^ (((token >> 2) & 1) << 1)) * ROW + chunk * 16;
    else if constexpr (D == 128) return (token ^ ((token >> 2) & 1)) * ROW + ((chunk ^ (token & 2)) * 16);
    else return token * ROW + ((chunk ^ (((token & 3) << 1) | ((token >> 2) & 1))) * 16);
  }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;  // nothing is read for 0 bytes: the place is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// the exponent of |v| as a float: 2^exponent <= |v| < 2^(exponent + 1); -127 for 0
__device__ __forceinline__ float exponent(float v) {
  return __uint_as_float(0x4b000000u | __float_as_uint(v) >> 23) - (8388608.0f + 127.0f);
}

constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;

struct RowsArgs {
  AttendArgs a;
  Join join;
};

template <int D, int NT>
struct Shared {
  static constexpr int R = 8 * NT;
  static constexpr int RING = kWarps * kStages * Stage<D>::BYTES;
  static constexpr int MERGE = kWarps * R * (D + 4) * 4;  // the ring's memory again
  static constexpr int BYTES = RING > MERGE ? RING : MERGE;
};

// Sums of a row tile as they leave a block: a thread holds 4 channels of each of N rows.
template <int D, int R>
struct Sums {
  static constexpr int N = (R * D / 4 + kWarps * 32 - 1) / (kWarps * 32);  // D = 64, R = 8: half of the threads hold one
  float4 v[N];
  static __device__ __forceinline__ int at(int e) { return threadIdx.x + e * kWarps * 32; }  // in fours
  static __device__ __forceinline__ bool some(int e) { return R * D / 4 % (kWarps * 32) == 0 || at(e) < R * D / 4; }
  static __device__ __forceinline__ int row(int e) { return at(e) / (D / 4) % R; }
  static __device__ __forceinline__ int channel(int e) { return at(e) % (D / 4) * 4; }
};

// The parts of a row tile (or of one group of its blocks) joined: the first at first_place, the
// others `step` blocks apart after `first`.  The statistics go through shared memory, so the loads of
// the parts do not wait for one another.
template <int D, int R>
__device__ __forceinline__ void join_parts(const Join& j, int first_place, int first, int count, int step,
                                           float (*weight)[R], float2* total, Sums<D, R>& sums) {
  auto place = [&](int i) { return i == 0 ? first_place : (first + i * step) * 2; };
  for (int x = threadIdx.x; x < count * R; x += kWarps * 32) {
    const int i = x / R, row = x - i * R;
    const float2 st = __ldcg(&j.stats[(int64_t)place(i) * R + row]);
    weight[i][row] = st.x;
    weight[count + i][row] = st.y;
  }
  __syncthreads();
  for (int row = threadIdx.x >> 5; row < R; row += kWarps) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY, sum = 0.0f;
    for (int i = lane; i < count; i += 32) m = fmaxf(m, weight[i][row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.0f : m;
    for (int i = lane; i < count; i += 32) {
      const float w = ex2(weight[i][row] - base);
      weight[i][row] = w;
      sum += w * weight[count + i][row];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) total[row] = make_float2(m, sum);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < Sums<D, R>::N; ++e) sums.v[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll(Sums<D, R>::N == 1 ? 16 : 8)
  for (int i = 0; i < count; ++i) {
    const float4* part = reinterpret_cast<const float4*>(j.parts + (int64_t)place(i) * R * D);
#pragma unroll
    for (int e = 0; e < Sums<D, R>::N; ++e) {
      if (!Sums<D, R>::some(e)) continue;
      const float4 x = __ldcg(part + Sums<D, R>::at(e));
      const float w = weight[i][Sums<D, R>::row(e)];
      sums.v[e].x += w * x.x;
      sums.v[e].y += w * x.y;
      sums.v[e].z += w * x.z;
      sums.v[e].w += w * x.w;
    }
  }
}

// Blocks on an SM: four (two where registers allow no more), three for row tiles of 16 with head_dim 64, which
// spilled with four (64 contexts of 700 tokens, 8 heads, 16 rows 29 us, was 34; 64 rows over 8,192 tokens 82, was 92).
constexpr int blocks_of(int dim, int nt) { return dim * nt > 128 ? 2 : (nt == 2 ? 3 : 4); }

template <int D, int NT, typename T>
__global__ void __launch_bounds__(kWarps * 32, blocks_of(D, NT)) attend_rows_kernel(const RowsArgs p) {
  const AttendArgs& a = p.a;
  using S = Stage<D>;
  constexpr int R = 8 * NT, KW = D / 32, VW = D / 64;  // rows of a tile; words of a key / value row's share of a lane
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t sh_scan[kWarps];
  __shared__ int sh_found[2];
  __shared__ Sequence sh_sequence;
  __shared__ int sh_last, sh_skipped;
  __shared__ float2 sh_stat[kWarps * R], sh_total[R], sh_origin[kWarps][R / 2];
  __shared__ float sh_weight[2 * kMostParts][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int heads = a.pool.kv_heads, page_size = a.pool.page_size;

  // ---- this block's share of the work: the steps of every sequence, row tile and head, and a few
  // for each of these items' start and end
  auto steps_of = [&](const Sequence& s) { return (s.length + kStep - 1) / kStep + kItemSteps; };
  auto items_of = [&](const Sequence& s) { return (int64_t)((s.count * a.group.d + R - 1) / R) * heads; };
  auto block_scan = [&](int64_t v, int64_t& total) {  // sum of v over the threads before this one
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh_scan[warp] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh_scan[w];
      total += sh_scan[w];
    }
    return before + x - v;
  };
  constexpr int64_t kUnits = ((int64_t)1 << 40) - 1;
  const int batch = (int)a.batch;
  if (threadIdx.x == 0) sh_skipped = 0;
  int64_t all = 0, items = 0, mine = 0, before = 0;
  Sequence seq{0, 0, 0, true};
  for (int b = 0; b < batch; b += kWarps * 32) {
    int64_t sum;
    mine = 0;
    if (b + (int)threadIdx.x < batch) {
      seq = sequence(a, b + threadIdx.x, blockIdx.x == 0);
      // units and items in one sum: no sequence within memory reaches these bounds
      mine = min(items_of(seq), (int64_t)1 << 20);
      mine = min(items_of(seq) * steps_of(seq), (int64_t)1 << 31) | mine << 40;
    }
    before = all + (block_scan(mine, sum) & kUnits);
    if (!seq.ok) sh_skipped = 1;
    all += sum & kUnits;
    items += sum >> 40;
    mine &= kUnits;
  }
  if (all > 0x7f000000) {  // starts that cross one another, or 2^36 tokens together: nothing is answered
    if (blockIdx.x == 0 && threadIdx.x == 0) flag(a.status, TANS_DEV_BAD_VALUE);
    zero_unanswered(a, D, blockIdx.x * (int64_t)(kWarps * 32) + threadIdx.x, (int64_t)gridDim.x * kWarps * 32, R, -1);
    return;
  }
  // With fewer items than half the blocks, each item has blocks of its own: as many as take `share` or
  // less each, its steps spread evenly over them.  These are at most all / share + items blocks.  Else the
  // blocks' shares follow one another across the items.  From here a sequence's extent is counted in
  // blocks or in units of work.
  const bool own = items < (int)gridDim.x / 2;
  const int sharers = own ? (int)(gridDim.x - items) : (int)gridDim.x;
  const int share = max(((int)all + sharers - 1) / sharers, kWarps + kItemSteps);
  auto extent_of = [&](const Sequence& s) { return own ? (steps_of(s) + share - 1) / share : steps_of(s); };
  if (own && batch <= kWarps * 32) {
    mine = threadIdx.x < batch ? items_of(seq) * extent_of(seq) : 0;
    before = block_scan(mine, all);
  } else if (own) {
    all = (int64_t)1 << 40;  // known when the end is reached
  }
  auto zero_rest = [&]() {
    zero_unowned<T>(a, D, blockIdx.x * (int64_t)(kWarps * 32) + threadIdx.x, (int64_t)gridDim.x * kWarps * 32);
    if (blockIdx.x == 0) {
      __syncthreads();
      if (sh_skipped) zero_unanswered(a, D, threadIdx.x, kWarps * 32, R, INT64_MAX);
    }
  };
  const int64_t start = (int64_t)blockIdx.x * (own ? 1 : share);
  if (start >= all) {
    zero_rest();
    return;
  }
  int u = (int)start;
  const int u_end = (int)min(all, start + (own ? 1 : share));
  if (threadIdx.x == 0) sh_found[0] = -1;
  __syncthreads();
  int64_t done = 0;
  for (int b = 0; b < batch; b += kWarps * 32) {
    if (batch > kWarps * 32) {  // more sequences than threads: once more from the start
      int64_t sum;
      mine = 0;
      if (b + (int)threadIdx.x < batch) {
        seq = sequence(a, b + threadIdx.x, false);
        mine = items_of(seq) * extent_of(seq);
      }
      before = done + block_scan(mine, sum);
      done += sum;
    }
    if (u >= before && u < before + mine) {
      sh_found[0] = b + threadIdx.x;
      sh_found[1] = (int)before;
      sh_sequence = seq;
    }
    if (u < done) break;
  }
  __syncthreads();
  int b = sh_found[0], b_first = sh_found[1];
  seq = sh_sequence;
  if (b < 0) {
    zero_rest();
    return;
  }

  uint8_t* ring = smem + warp * kStages * S::BYTES;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);

  // this lane's places in a step: what it copies (of the first 16 tokens), and what it reads.  Tokens
  // 8 and 16 further lie 8 and 16 rows further.
  int copy_at[S::COPIES], key_at[KW > 4 ? 2 : 1], value_at[2];
#pragma unroll
  for (int i = 0; i < S::COPIES; ++i) copy_at[i] = S::place((i * 32 + lane) / S::CHUNKS, (i * 32 + lane) % S::CHUNKS);
  const int tok = (g >> 1) + (g & 1) * 4;  // rows g and g + 8 of the score's product are tokens tok and tok + 8
  if constexpr (KW >= 4) {
#pragma unroll
    for (int i = 0; i < KW / 4; ++i) key_at[i] = S::K + S::place(tok, t * (KW / 4) + i);
  } else {
    key_at[0] = S::K + S::place(tok, t >> 1) + (t & 1) * 8;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // tokens t + 4 j, t + 8 + 4 j
    const int c = VW == 4 ? g : (VW == 2 ? g >> 1 : g >> 2), in = VW == 4 ? 0 : (VW == 2 ? (g & 1) * 8 : (g & 3) * 4);
    value_at[j] = S::V + S::place(t + 4 * j, c) + in;
  }

  while (u < u_end) {
    while (u >= b_first + items_of(seq) * extent_of(seq)) {  // sequences without queries have no extent
      b_first += (int)(items_of(seq) * extent_of(seq));
      ++b;
      seq = sequence(a, b, false);
    }
    const int extent = extent_of(seq), steps = steps_of(seq) - kItemSteps;
    const int item = (u - b_first) / extent, item_first = b_first + item * extent;
    const int u_next = min(item_first + extent, u_end);
    const int step0 = own ? (int)((int64_t)(u - item_first) * steps / extent) : max(0, u - item_first - kItemSteps);
    const int step1 = own ? (int)((int64_t)(u_next - item_first) * steps / extent) : max(0, u_next - item_first - kItemSteps);
    const int tile = a.kv_heads.div(item), head = item - tile * heads;
    const int row0 = tile * R, rows = min(R, seq.count * (int)a.group.d - row0);

    // ---- this lane's quarters of the query rows, row g of each 8; they are turned to float16 below
    uint4 raw[NT][D / 32];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) raw[n][c] = make_uint4(0, 0, 0, 0);
      if (n * 8 + g < rows) {
        const int r = row0 + n * 8 + g, i = a.group.div(r), h = head * a.group.d + (r - i * a.group.d);
        const T* src = static_cast<const T*>(a.q) + (seq.start + i) * a.q_ts + h * a.q_hs + t * (D / 4);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          if (a.vec) {
            raw[n][c] = *reinterpret_cast<const uint4*>(src + c * 8);
          } else {
            const uint16_t* u = reinterpret_cast<const uint16_t*>(src + c * 8);
            raw[n][c] = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16,
                                   u[6] | (uint32_t)u[7] << 16);
          }
        }
      }
    }

    // ---- steps of this warp: step0 + warp, + kWarps, ...; kStages - 1 of them on their way
    uint32_t known = 0;  // two bits a step in flight, the newest lowest: the group's page is one of the pool
    const uint32_t side_rows = (uint32_t)heads * page_size;  // from a page's keys to its values, and half a page (< 2^31)
    const uint8_t* head_codes = a.pool.codes + (int64_t)head * page_size * S::ROW + lane * 16;
    const uint32_t* head_params =
        a.pool.params + ((lane >= 4 ? heads : 0) + (int64_t)head) * page_size + (lane & 3) * 4;
    const int32_t* table = a.pages + (int64_t)b * a.max_pages;
    // the page and the place in it of the next step's first token; from step to step they grow alike
    int next = step0 + warp;
    int at = a.page_size.div(next * kStep), first = next * kStep - at * page_size;
    const int more_pages = a.page_size.div(kWarps * kStep), more_tokens = kWarps * kStep - more_pages * page_size;
    // its pages are looked up a step ahead; -1: no tokens there
    int page[2];
    auto look_up = [&]() {
      int h_at = at, h_first = first;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        page[h] = -1;
        if (next < step1 && next * kStep + h * 16 < seq.length) page[h] = __ldg(table + h_at);
        h_first += 16;
        if (h_first == page_size) {
          h_first = 0;
          ++h_at;
        }
      }
    };
    look_up();
    auto fetch = [&](int slot) {
      uint32_t bits = 0;
      if (next < step1) {
        const uint32_t base = ring_at + slot * S::BYTES;
        int h_first = first;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool there = (unsigned)page[h] < (unsigned)a.pool.num_pages;
          if (!there && lane == 0 && next * kStep + h * 16 < seq.length) flag(a.status, TANS_DEV_BAD_INDEX);
          if (there) bits |= 1u << h;
          const uint64_t page_row = (uint64_t)(there ? page[h] : 0) * (2 * side_rows);
          const uint8_t* ks = head_codes + (page_row + h_first) * S::ROW;
          const uint8_t* vs = ks + (uint64_t)side_rows * S::ROW;
#pragma unroll
          for (int i = 0; i < S::COPIES; ++i) {
            cp16(base + S::K + h * 16 * S::ROW + copy_at[i], ks + i * 512, there);
            cp16(base + S::V + h * 16 * S::ROW + copy_at[i], vs + i * 512, there);
          }
          if (lane < 8)  // keys' parameters, then values'
            cp16(base + S::KP + (lane >> 2) * kStep * 4 + h * 64 + (lane & 3) * 16,
                 head_params + page_row + h_first, there);
          h_first += 16;
          if (h_first == page_size) h_first = 0;
        }
        next += kWarps;
        at += more_pages;
        first += more_tokens;
        if (first >= page_size) {
          first -= page_size;
          ++at;
        }
        look_up();
      }
      known = known << 2 | bits;
      cp_commit();
    };
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(i);

    // ---- the queries: column g of each 8 is row g; a lane's channels are the t-th quarter
    uint32_t qf[NT][KW][4];
    float fac[NT][2], shift[NT][2];  // of columns 2t and 2t + 1: score = (acc * s) * fac + o * shift
    int seen[NT][2];                 // tokens that the columns' queries see
    uint32_t large[NT];              // bit 8 t + 4 c: a score lacks 2^24
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[D / 4];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint32_t v[4] = {raw[n][c].x, raw[n][c].y, raw[n][c].z, raw[n][c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Half2<T>::unpack(v[e]);
          x[c * 8 + 2 * e] = f.x;
          x[c * 8 + 2 * e + 1] = f.y;
        }
      }
      float top = 0.0f, sum = 0.0f;  // 2^-10 of the sum: it may pass float's range
#pragma unroll
      for (int c = 0; c < D / 4; ++c) {
        top = fmaxf(top, fabsf(x[c]));
        sum = fmaf(x[c], 0.0009765625f, sum);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      const int e = 13 - max(-113, min(127, (int)(__float_as_uint(top) >> 23) - 127));  // the row times 2^e is under 2^14
      // the score's factors, 2^(24 - e), may pass float's range for large queries: those lack 2^24 until the end
      const bool over = e < -100;
      large[n] = __ballot_sync(0xffffffffu, over);
      const float up = pow2(e), up16 = pow2(e - 4);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        // the codes of a word pair up as (0, 4), (1, 5), (2, 6), (3, 7); the odd ones come 16 times too large
        qf[n][w][0] = Half2<__half>::pack(x[8 * w] * up, x[8 * w + 4] * up);
        qf[n][w][1] = Half2<__half>::pack(x[8 * w + 1] * up16, x[8 * w + 5] * up16);
        qf[n][w][2] = Half2<__half>::pack(x[8 * w + 2] * up, x[8 * w + 6] * up);
        qf[n][w][3] = Half2<__half>::pack(x[8 * w + 3] * up16, x[8 * w + 7] * up16);
      }
      const float f = a.scale_log2 * pow2(over ? -e : 24 - e), sh = a.scale_log2 * (over ? 0x1p-14f : 1024.0f) * sum;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        fac[n][c] = __shfl_sync(0xffffffffu, f, (2 * t + c) * 4);
        shift[n][c] = __shfl_sync(0xffffffffu, sh, (2 * t + c) * 4);
        const int col = n * 8 + 2 * t + c;
        const int i = a.group.div(row0 + col);
        seen[n][c] = col >= rows ? 0 : (a.causal ? min(seq.length, seq.length - seq.count + i + 1) : seq.length);
      }
    }
    // every live row sees the tokens under `full`
    const int full = a.causal ? seq.length - seq.count + a.group.div(row0) + 1 : seq.length;

    // Some scores lack 2^24, or have an origin: all steps go the longer way.
    bool apart = false;
    float2* const origin = sh_origin[warp];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      apart |= large[n] != 0;
      if (g == 0) origin[n * 4 + t] = make_float2(0.0f, 0.0f);
    }
    __syncwarp();
    // of columns 2t and 2t + 1: m and Y as above, the sums of the weights and of their offsets in 2^R, the
    // products in 2^Y
    float m[NT][2], Y[NT][2], l[NT][2], off[NT][2], acc[NT][D / 16][4], ones[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[n][c] = -INFINITY;
        Y[n][c] = kNone;
        l[n][c] = off[n][c] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.0f;
      ones[n][0] = ones[n][1] = ones[n][2] = ones[n][3] = 0.0f;
    }

    int slot = 0;
    for (int step = step0 + warp; step < step1; step += kWarps) {
      cp_wait<kStages - 2>();
      __syncwarp();
      const uint32_t bits = known >> (2 * (kStages - 2));
      fetch(slot == 0 ? kStages - 1 : slot - 1);
      const uint8_t* st = ring + slot * S::BYTES;
      slot = slot == kStages - 1 ? 0 : slot + 1;

      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t k0[KW], k1[KW];
        if constexpr (KW >= 4) {
#pragma unroll
          for (int i = 0; i < KW / 4; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(st + key_at[i] + h * 16 * S::ROW);
            const uint4 y = *reinterpret_cast<const uint4*>(st + key_at[i] + (h * 16 + 8) * S::ROW);
            k0[4 * i] = x.x; k0[4 * i + 1] = x.y; k0[4 * i + 2] = x.z; k0[4 * i + 3] = x.w;
            k1[4 * i] = y.x; k1[4 * i + 1] = y.y; k1[4 * i + 2] = y.z; k1[4 * i + 3] = y.w;
          }
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(st + key_at[0] + h * 16 * S::ROW);
          const uint2 y = *reinterpret_cast<const uint2*>(st + key_at[0] + (h * 16 + 8) * S::ROW);
          k0[0] = x.x; k0[1] = x.y;
          k1[0] = y.x; k1[1] = y.y;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const uint32_t x = k0[w], y = k1[w], x8 = x >> 8, y8 = y >> 8;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma(s[h][n], x & kLow, y & kLow, x & kHigh, y & kHigh, qf[n][w][0], qf[n][w][1]);
            mma(s[h][n], x8 & kLow, y8 & kLow, x8 & kHigh, y8 & kHigh, qf[n][w][2], qf[n][w][3]);
          }
        }
      }

      // Scores to weights.  `masked` steps hold tokens past the end, of unknown pages or past a query:
      // their scores are -inf and their parameters, which may be anything, count nowhere.
      uint32_t wf[2][NT][2];
      auto weigh = [&](auto masked_) {
        constexpr bool masked = decltype(masked_)::value;
        const uint32_t* kp = reinterpret_cast<const uint32_t*>(st + S::KP) + tok;
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(st + S::VP) + tok;
        float sv[4], ov[4], top[NT][2];
        bool in[4];
#pragma unroll
        for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
        float big = 0.0f;  // the largest size
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // j: group j / 2, row g or g + 8
          const uint32_t kw = kp[8 * j], vw = vp[8 * j];
          const float sk = scale_of(kw), ok = offset_of(kw);
          sv[j] = scale_of(vw);
          ov[j] = fmaf(7.5f, sv[j], offset_of(vw));
          const int token = step * kStep + tok + 8 * j;
          in[j] = !masked || (token < seq.length && (bits >> (j >> 1) & 1));
          const float size = fmaxf(fabsf(sv[j]), fabsf(ov[j]));
          big = fmaxf(big, in[j] ? size : 0.0f);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float& x = s[j >> 1][n][(j & 1) * 2 + c];
              x = fmaf(x * sk, fac[n][c], ok * shift[n][c]);
              if (masked && (large[n] >> (8 * t + 4 * c) & 1)) x *= 16777216.0f;
              if (masked && !(in[j] && token < seen[n][c])) x = -INFINITY;
              top[n][c] = fmaxf(top[n][c], x);
            }
        }
        const float reach = exponent(big) - kRoom;
        // scores are as they are until their origin, which may move, is taken off below
        float from[NT][2];
        bool move = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            from[n][c] = !masked || !apart ? 0.0f : (c ? origin[n * 4 + t].y : origin[n * 4 + t].x);
            const float x = top[n][c] - from[n][c];
            move |= x > m[n][c] + kSlack || x + reach > Y[n][c];
          }
        if (__any_sync(0xffffffffu, move)) {
          // the columns' reductions side by side: the largest scores, then the largest products
          float now[NT][2], y[NT][2];
          auto across = [&](float (&v)[NT][2]) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1)
#pragma unroll
              for (int i = 0; i < 2 * NT; ++i) v[i >> 1][i & 1] = fmaxf(v[i >> 1][i & 1], __shfl_xor_sync(0xffffffffu, v[i >> 1][i & 1], o));
          };
#pragma unroll
          for (int i = 0; i < 2 * NT; ++i) now[i >> 1][i & 1] = top[i >> 1][i & 1];
          across(now);
          bool far[NT][2], some_far = false;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float x = now[n][c] - from[n][c];
              far[n][c] = x > m[n][c] + kSlack && fabsf(x) > kFar;
              some_far |= far[n][c];
            }
          if (__any_sync(0xffffffffu, some_far)) {  // their origin becomes the largest score itself
            apart = true;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if (!far[n][c]) continue;
                const float by = now[n][c] - from[n][c];
                Y[n][c] = m[n][c] == -INFINITY ? kNone : Y[n][c] - by;
                m[n][c] -= by;
                from[n][c] = now[n][c];
                if (g == 0) reinterpret_cast<float*>(origin)[(n * 4 + t) * 2 + c] = now[n][c];
              }
            __syncwarp();
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              now[n][c] -= from[n][c];
              now[n][c] = now[n][c] > m[n][c] + kSlack ? now[n][c] : m[n][c];
              y[n][c] = -INFINITY;
#pragma unroll
              for (int j = 0; j < 4; ++j)  // a token that the row does not see is at -inf, whatever its size
                y[n][c] = fmaxf(y[n][c], s[j >> 1][n][(j & 1) * 2 + c] - from[n][c] + exponent(fmaxf(fabsf(sv[j]), fabsf(ov[j]))));
            }
          across(y);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float Y_now = y[n][c] > Y[n][c] + kRoom ? y[n][c] - (kRoom - kSlack) : Y[n][c];
              if (now[n][c] != -INFINITY) Y_now = fminf(fmaxf(Y_now, now[n][c] - kDeepest), now[n][c] + kHighest);
              if (m[n][c] != -INFINITY) {  // nothing is kept before the first token
                const float keep = ex2(fminf(m[n][c], Y[n][c]) - fminf(now[n][c], Y_now)), both = ex2(Y[n][c] - Y_now);
                l[n][c] *= keep;
                off[n][c] *= keep;
                ones[n][c] *= both;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                  acc[n][i][c] *= both;
                  acc[n][i][c + 2] *= both;
                }
              }
              m[n][c] = now[n][c];
              Y[n][c] = Y_now;
            }
        }
        if (apart) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i >> 2][n][i & 3] -= from[n][i & 1];
        }
        float base[NT][2], less[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float unit = fminf(m[n][c], Y[n][c]);
            base[n][c] = m[n][c] == -INFINITY ? 0.0f : unit;
            less[n][c] = ex2(unit - Y[n][c]);  // 1 unless values are larger than 2^6
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float w[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float x = s[j >> 1][n][(j & 1) * 2 + c];
              const float e = ex2(x - base[n][c]);
              const bool hidden = masked && x == -INFINITY;
              l[n][c] += e;
              w[c] = hidden ? 0.0f : e * (sv[j] * less[n][c]);
              off[n][c] = hidden ? off[n][c] : fmaf(e, ov[j], off[n][c]);
            }
            wf[j >> 1][n][j & 1] = transpose8(Half2<__half>::pack(w[0], w[1]));
          }
        }
      };
      if ((bits & 3u) == 3u && (step + 1) * kStep <= full && !apart) weigh(std::false_type{});
      else weigh(std::true_type{});

      // ---- values
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[4][VW];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint8_t* src = st + value_at[j & 1] + (h * 16 + (j & 2) * 4) * S::ROW;
          if constexpr (VW == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(src);
            v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
          } else if constexpr (VW == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            v[j][0] = x.x; v[j][1] = x.y;
          } else {
            v[j][0] = *reinterpret_cast<const uint32_t*>(src);
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // channels 4 half .. 4 half + 3 of the word: tokens (t, t + 4) and (t + 8, t + 12)
            uint32_t x = __byte_perm(v[0][w], v[1][w], half ? 0x7632 : 0x5410);
            uint32_t y = __byte_perm(v[2][w], v[3][w], half ? 0x7632 : 0x5410);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma(acc[n][w * 4 + half * 2 + q], x & kLow, x & kHigh, y & kLow, y & kHigh, wf[h][n][0], wf[h][n][1]);
              x >>= 8;
              y >>= 8;
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma(ones[n], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, wf[h][n][0], wf[h][n][1]);
      }
    }
    cp_wait<0>();

    // ---- join the warps: sums in shared memory (the rings' memory)
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);  // [warp][row][D + 4]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
          off[n][c] += __shfl_xor_sync(0xffffffffu, off[n][c], o);
        }
        const int row = n * 8 + 2 * t + c;
        // all in 2^m
        const bool none = m[n][c] == -INFINITY;
        const float back = none ? 0.0f : ex2(Y[n][c] - m[n][c]), low = none ? 1.0f : ex2(fminf(Y[n][c] - m[n][c], 0.0f));
        const float2 from = origin[n * 4 + t];
        l[n][c] *= low;
        off[n][c] *= low;
        float* dst = so + (warp * R + row) * (D + 4) + g * (D / 8);
        const float mid = 7.5f * ones[n][c];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          dst[2 * i] = fmaf(fmaf(acc[n][i][c], 16777216.0f, -mid), back, off[n][c]);
          dst[2 * i + 1] = fmaf(fmaf(acc[n][i][c + 2], 1048576.0f, -mid), back, off[n][c]);
        }
        if (g == 0) sh_stat[warp * R + row] = make_float2(m[n][c] + (c ? from.y : from.x), l[n][c]);
      }
    __syncthreads();

    using Part = Sums<D, R>;
    Part sums;
#pragma unroll
    for (int e = 0; e < Part::N; ++e) {
      const int row = Part::row(e), d = Part::channel(e);
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh_stat[w * R + row].x);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 st = sh_stat[w * R + row];
        const float k = ex2(st.x - base);
        const float4 x = *reinterpret_cast<const float4*>(so + (w * R + row) * (D + 4) + d);
        sum += k * st.y;
        v.x += k * x.x;
        v.y += k * x.y;
        v.z += k * x.z;
        v.w += k * x.w;
      }
      sums.v[e] = v;
      if (d == 0 && Part::some(e)) sh_total[row] = make_float2(top, sum);
    }
    __syncthreads();  // the rings may be filled again

    // ---- whole here, or joined with the other blocks' parts
    bool whole = u == item_first && u_next == item_first + extent;
    if (!whole) {
      const Join& j = p.join;
      const int c0 = own ? item_first : item_first / share;
      const int c1 = own ? item_first + extent - 1 : (item_first + extent - 1) / share;
      auto leave = [&](int place) {
#pragma unroll
        for (int e = 0; e < Part::N; ++e)
          if (Part::some(e)) reinterpret_cast<float4*>(j.parts + (int64_t)place * R * D)[Part::at(e)] = sums.v[e];
        if (threadIdx.x < R) j.stats[(int64_t)place * R + threadIdx.x] = sh_total[threadIdx.x];
        __threadfence();
        __syncthreads();
      };
      auto last_of = [&](int level, int place, int expected) {
        if (threadIdx.x == 0) sh_last = arrive(j.arrivals + level * kMostBlocks * 2 + place, expected);
        __syncthreads();
        const bool last = sh_last != 0;
        __syncthreads();
        __threadfence();
        return last;
      };
      const int me = blockIdx.x;
      leave(me * 2 + (me == c0));
      const int f0 = c0 + (me - c0) / kFan * kFan, f1 = min(c1, f0 + kFan - 1);  // this block's group
      const int place = f0 * 2 + (f0 == c0);
      whole = f1 == f0 || last_of(0, place, f1 - f0 + 1);
      if (whole && f1 > f0) join_parts<D, R>(j, place, f0, f1 - f0 + 1, 1, sh_weight, sh_total, sums);
      if (whole && (f0 != c0 || f1 != c1)) {  // the groups
        if (f1 > f0) leave(place);
        const int groups = (c1 - c0) / kFan + 1;
        whole = last_of(1, c0 * 2 + 1, groups);
        if (whole) join_parts<D, R>(j, c0 * 2 + 1, c0, groups, kFan, sh_weight, sh_total, sums);
      }
    }
    if (whole) {
#pragma unroll
      for (int e = 0; e < Part::N; ++e) {
        const int row = Part::row(e), d = Part::channel(e);
        if (row < rows && Part::some(e)) {
          const int r = row0 + row, i = a.group.div(r), h = head * a.group.d + (r - i * a.group.d);
          const int64_t o = (int64_t)(seq.start + i) * a.q_heads + h;
          const float2 st = sh_total[row];
          const float k = st.y == 0.0f ? 0.0f : 1.0f / st.y;
          uint2 w;
          w.x = Half2<T>::pack(sums.v[e].x * k, sums.v[e].y * k);
          w.y = Half2<T>::pack(sums.v[e].z * k, sums.v[e].w * k);
          *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + o * D + d) = w;
          if (a.lse && d == 0) a.lse[o] = st.y == 0.0f ? -INFINITY : (st.x + log2f(st.y)) * 0.69314718055994531f;
        }
      }
      __syncthreads();  // the totals may be written again
    }
    u = u_next;
  }
  zero_rest();
}

// Blocks that an SM holds at once, found once for each device (a kernel's attributes are the device's).
template <int D, int NT, typename T>
int blocks_per_sm() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    constexpr int bytes = Shared<D, NT>::BYTES;
    if (cudaFuncSetAttribute(attend_rows_kernel<D, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
            cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attend_rows_kernel<D, NT, T>, kWarps * 32, bytes) !=
            cudaSuccess)
      return 0;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int D, int NT, typename T>
int launch(const AttendArgs& a, void* workspace, cudaStream_t s) {
  const int per_sm = blocks_per_sm<D, NT, T>();
  if (per_sm < 1) return TANS_E_CUDA;
  const int blocks = std::min(kMostBlocks, per_sm * sm_count());
  const Join j = Join::in(workspace, 8 * NT);
  attend_rows_kernel<D, NT, T><<<blocks, kWarps * 32, Shared<D, NT>::BYTES, s>>>(RowsArgs{a, j});
  note_launch();
  return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
}

}  // namespace

// Row tiles of 16 instead of 8.  The cache is read half as often, and a step costs about 1.3 times as much:
// at 9 rows or more it pays (16 contexts of 8,192 tokens, 4 heads of 128, 16 rows: 39 against 49 us, of 64: 33
// against 37; 64 contexts of 700 tokens, 8 heads of 128: 43 both), but not for head_dim 256, whose sums then do
// not fit the registers.
static bool wide_tiles(int head_dim, int64_t max_rows) { return head_dim <= 128 && max_rows > 8; }

size_t attend_rows_workspace(int head_dim, int64_t max_rows) {
  const int64_t rows = wide_tiles(head_dim, max_rows) ? 16 : 8;
  return align_up(Join::bytes(rows, head_dim));
}

int launch_attend_rows(const AttendArgs& a, int dtype, int64_t max_rows, void* workspace, cudaStream_t s) {
  auto by_rows = [&](auto d, auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int D = decltype(d)::value;
    if constexpr (D <= 128) {
      if (wide_tiles(D, max_rows)) return launch<D, 2, T>(a, workspace, s);
    }
    return launch<D, 1, T>(a, workspace, s);
  };
  auto by_dim = [&](auto* t) {
    return a.pool.head_dim == 64    ? by_rows(std::integral_constant<int, 64>{}, t)
           : a.pool.head_dim == 128 ? by_rows(std::integral_constant<int, 128>{}, t)
                                    : by_rows(std::integral_constant<int, 256>{}, t);
  };
  return dtype == TANS_BF16 ? by_dim(static_cast<__nv_bfloat16*>(nullptr)) : by_dim(static_cast<__half*>(nullptr));
}

}  // namespace kv4
}  // namespace tans
