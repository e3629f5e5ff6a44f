// kv4_attend_prompt.cu -- attention over the 4-bit cache when many query rows share a key/value head
// (whole prompts, chunks of them, many drafted tokens or very wide groups): bound by arithmetic, so
// both products run on tcgen05 with their accumulators in tensor memory.
//
// A block takes 128 (head_dim 256) or 2 x 128 query rows of one key/value head, row r being head
// r mod group of query r / group, and walks over the tokens 128 at a time:
//   softmax warps   4 for each 128 rows, a thread for a row: they read the scores S from tensor
//                   memory, keep the row's running maximum and sum, and put the weights P back over S
//                   as float16;
//   unpacking warps 4, a thread for a token: its codes become float16 c * s + o in shared memory, in
//                   the swizzled rows that the tensor cores read (keys K-major; the same rows of
//                   values are an MN-major operand, so nothing is transposed);
//   one warp        issues S = Q K^T (both from shared memory) and O += P V (P from tensor memory).
// Scores come 64 tokens at a time into two places of each tile in turn, so the softmax of one half step
// runs while the products of the half steps around it do, and waits for none of them.
//
// A block goes on to the next of its row tiles by itself: the unpacking warps are then already there,
// and the next queries come while the last results leave.
//
// Where there are fewer such row tiles than SMs, several blocks share the tokens of each, leave their
// sums in the workspace, and the last of them joins them in the order of the tokens.
//
// All operands are float16 brought into range by powers of two: a query row by its own, the keys and the
// values of a step by one each.  Rows that differ by over 2^5 need another conversion (1 % more time if all steps
// have such); rows that differ by more than 2^11 (keys) or 2^8 (values) would lose bits of themselves or of the weights:
// a step with such rows is "wide", and there each row has its own factor, which the softmax warps put into
// its scores and weights, in some seven times the time.  So the rounding is 2^-11
// of each key, each value and each weight, whatever the sizes of other tokens, of those that are hidden
// from a query too; sums are float.
//
// A query row's weights are 2^(x - m - d) for the score x, its running maximum m and a power of two d of
// its own over the step's: it follows the largest product of a weight and a value's size that the row sees, and
// leaves it at 2^6 when it moves, which it does (and O is rescaled) when a product passes it by 2^14.  The
// sum of the softmax is 2^(x - m), which m follows when a score passes it by over 8.  Scores are fused into
// x - (m + d); where |m| passes 2^10 they are rounded first and m is taken from them, token by token as in a
// wide step: the product's rounding would otherwise be a factor of the weight, past float's range from 2^30.
//
// Measured: 4 packed prompts of 1,143 to 3,500 tokens (32 query and 8 key/value heads of 128, 166 GFLOP) 236
// us, 703 TFLOP/s; 511 queries over 32,749 tokens (16 and 4 heads of 64, 68 GFLOP) 169 us, 402 TFLOP/s.  With one power
// of two for all values so far and none for single rows these took 228 and 161 us on the same GPU, and a value 2^16
// times larger in a step, seen or not, left other queries' answers a fifth wrong.  Such prompts with one row in
// 16 2^4 times larger: 263 us where others take 260; 2^14 times: 1,860 (every step wide); scores past 2^10: 1,210.
// A half step takes about 2,000 cycles, in which the products are busy for 1,280 (head_dim 128), 2^x for 1,024
// and the instructions' issue for 900 a scheduler: leaving out any one of them, or the unpacking, in a copy
// took 2 to 4 % off (17 % for 2^x at head_dim 64), so it is the latency of all of them together.  Steps of 128
// tokens whose softmax waits for its own products took 261 us where half steps took 243; without the blocks'
// going on by themselves 243 against 233.
#include "kv4_attend.cuh"
#include "launch.cuh"
#include "rans_host.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace tans {
namespace kv4 {
namespace {

constexpr int kTile = 128;  // rows of a tile, tokens of a step
constexpr int kHalf = 64;   // tokens of a half step
constexpr float kSlack = 8.0f;  // by which a score may pass the running maximum
constexpr float kRoom = 14.0f;  // largest exponent of a weight
constexpr float kFar = 1024.0f; // a maximum from here on is taken from the rounded scores: m + d would be rounded, too
constexpr int kInfos = 4;   // steps whose factors are kept: the unpacking warps run at most 2 ahead
constexpr int kTries = 1 << 20;  // of the last wait

template <int D>
struct Plan {
  static constexpr int TILES = D == 256 ? 1 : 2;   // row tiles of a block
  static constexpr int STAGES = D == 256 ? 1 : 2;  // steps of unpacked keys and values
  // a warpgroup for each row tile, two for unpacking, one for issuing (of which one warp works)
  static constexpr int UNPACK = 4 * TILES, ISSUE = UNPACK + 8, WARPS = ISSUE + 4;
  // Registers of a thread, moved to the groups that need more.  What the groups' threads hold together
  // must not be more than the launch gave them.
  static constexpr int LAUNCH_REGS = TILES == 2 ? 96 : 128;
  static constexpr int SOFTMAX_REGS = TILES == 2 ? 144 : 240, UNPACK_REGS = TILES == 2 ? 72 : 112,
                       ISSUE_REGS = TILES == 2 ? 48 : 40;
  static_assert(UNPACK * SOFTMAX_REGS + 8 * UNPACK_REGS + 4 * ISSUE_REGS <= WARPS * LAUNCH_REGS, "a wait without end");
  static constexpr int BLOCK = kTile * 128;        // bytes of 64 channels of 128 rows
  static constexpr int ROWS = BLOCK * (D / 64);    // bytes of 128 rows
  static constexpr int Q = 0, K = ROWS * TILES, V = K + ROWS * STAGES, END = V + ROWS * STAGES;
  // over half of an SM's shared memory even for head_dim 64: one block on an SM, which takes all of
  // its tensor memory
  static constexpr int BYTES = (END > 120 * 1024 ? END : 120 * 1024) + 1024;
  static constexpr int S_COLUMNS = 128;
  static constexpr int O = S_COLUMNS * TILES;  // first column of O
};

// The blocks that share a row tile's tokens, and where they leave their sums.
struct Split {
  int splits;     // blocks for each row tile and head
  int* arrivals;  // one for each of these; without a split: pieces of work given out, blocks that have no more
  float2* stats;  // [row tile and head][splits][rows]: maximum (a power of two's exponent) and sum
  float4* parts;  // [row tile and head][splits][dim / 4][rows]
};
constexpr int kLeastSteps = 4;  // that a block takes, if there are as many

struct alignas(16) Info {  // of a step, from the unpacking warps to the softmax warps
  float key0, key1;    // the product of these undoes the keys' power of two (in a wide step each key has its own)
  float value_shift;   // values are 2^value_shift times too large
  uint8_t special[4];  // 1: 32 tokens have one in the following; 2: the step is wide
  uint32_t hidden[4], bad[4];  // tokens that no row sees, and those whose value is not finite
};

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_of(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_of(bar)) : "memory");
}
// A bounded wait.  One that runs out is recorded in `stalled`; waits after that return at once, so the
// block comes to its end (with values that are not valid) and frees its tensor memory.  Warps leave their
// loops early then, each as a whole (`stalled` is read by a vote where it decides); warps that meet at a named
// barrier later on decide together, at that barrier (any_of), so that none waits there for one that has left.
// What a wait was to protect is not written after one that ran out where others take addresses from it (the
// queue).
__device__ __forceinline__ void bar_wait(uint64_t* bar, uint32_t parity, int tries, volatile int* stalled) {
  const uint32_t at = smem_of(bar);
  uint32_t done;
  asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.b32 %0, 1, 0, p;\n}\n"
               : "=r"(done)
               : "r"(at), "r"(parity)
               : "memory");
  if (done) return;
  for (int i = 0; i < tries; ++i) {
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(at), "r"(parity), "r"(1000)  // a microsecond each
        : "memory");
    if (done) return;
    if (*stalled) return;
  }
  *stalled = 1;
}

// A barrier of `threads` that tells all of them whether `one` is true for any.
template <int BARRIER, int THREADS>
__device__ __forceinline__ bool any_of(bool one) {
  uint32_t any;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 q, %1, 0;\nbar.red.or.pred p, %2, %3, q;\nselp.b32 %0, 1, 0, p;\n}\n"
               : "=r"(any)
               : "r"((uint32_t)one), "n"(BARRIER), "n"(THREADS)
               : "memory");
  return any != 0;
}

// true for one thread of the warp
__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_of(bar))
               : "memory");
}

// Shared memory operand: rows of 128 bytes in the 128-byte swizzle, 8 rows to 1024 bytes; `leading` is
// the distance of the next 64 values of an MN-major operand.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t leading) {
  return (uint64_t)((at & 0x3ffff) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// float16 operands, float accumulator, 128 rows, n columns
__host__ __device__ constexpr uint32_t instruction(int n, bool b_mn_major) {
  return 1u << 4 | (b_mn_major ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kTile >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool more) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)more)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool more) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)more)
      : "memory");
}

// Two float products and sums in one instruction.
__device__ __forceinline__ uint64_t pair(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)), "l"(pair(c)));
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)));
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}

#define TANS_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define TANS_W4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
// 32 columns of this warp's 32 rows: a thread has its row's
__device__ __forceinline__ void load32(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : TANS_R4(r, 0), TANS_R4(r, 4), TANS_R4(r, 8), TANS_R4(r, 12), TANS_R4(r, 16), TANS_R4(r, 20), TANS_R4(r, 24),
        TANS_R4(r, 28)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void load16(uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : TANS_R4(r, 0), TANS_R4(r, 4), TANS_R4(r, 8), TANS_R4(r, 12)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void store16(const uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::TANS_W4(
          r, 0),
      TANS_W4(r, 4), TANS_W4(r, 8), TANS_W4(r, 12), "r"(at)
      : "memory");
}
__device__ __forceinline__ void store8(const uint32_t (&r)[8], uint32_t at) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::TANS_W4(r, 0), TANS_W4(r, 4),
               "r"(at)
               : "memory");
}
__device__ __forceinline__ void loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
#define TANS_RW4(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3])
// no use of these registers comes before this place (the wait that the loads into them need)
__device__ __forceinline__ void hold(uint32_t (&r)[16]) {
  asm volatile("" : TANS_RW4(r, 0), TANS_RW4(r, 4), TANS_RW4(r, 8), TANS_RW4(r, 12));
}
__device__ __forceinline__ void hold(uint32_t (&r)[32]) {
  asm volatile(""
               : TANS_RW4(r, 0), TANS_RW4(r, 4), TANS_RW4(r, 8), TANS_RW4(r, 12), TANS_RW4(r, 16), TANS_RW4(r, 20),
                 TANS_RW4(r, 24), TANS_RW4(r, 28));
}
__device__ __forceinline__ void stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 8 codes as float16 values c * s + o, in the order 0, 4, 1, 5, 2, 6, 3, 7.  The bits of c in the low four bits
// of a half are the subnormal c * 2^-24, in the next four c * 2^-20, and the factors are `low` = s * 2^24 and `high` =
// s * 2^20.  FULL: all are brought to bits 6 to 9, c * 2^-18, and the factor `low` is s * 2^18, which leaves 6 more
// powers of two to the rows' sizes.  The product is exact either way, so a value is rounded once.
template <bool FULL>
__device__ __forceinline__ uint4 unpack8(uint32_t w, __half2 low, __half2 high, __half2 o) {
  auto value = [&](uint32_t c, __half2 s) {
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&c), s, o);
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  if constexpr (FULL)
    return make_uint4(value(w << 6 & 0x03c003c0u, low), value(w << 2 & 0x03c003c0u, low), value(w >> 2 & 0x03c003c0u, low),
                      value(w >> 6 & 0x03c003c0u, low));
  const uint32_t x = w >> 8;
  return make_uint4(value(w & 0x000f000fu, low), value(w & 0x00f000f0u, high), value(x & 0x000f000fu, low),
                    value(x & 0x00f000f0u, high));
}

// v * 2^n, n in -252 .. 254
__device__ __forceinline__ float scaled(float v, int n) { return v * pow2(n >> 1) * pow2(n - (n >> 1)); }

__device__ __forceinline__ bool finite_row(uint32_t p) {
  return fabsf(scale_of(p)) < INFINITY && fabsf(offset_of(p)) < INFINITY;  // neither for NaN
}
// The size of a row's values as an exponent field, 0 for a row that is zero or not finite.  2^(kReach - size)
// brings the values under 2^-7 and, since 7.5 scales are no more than the largest value, the scale times 2^24
// under 2^15.
constexpr int kReach = 119, kMostShift = 113;
// Rows of a step that are so much smaller than its largest are at 2^-13 still, where float16 rounds to 2^-25.  Keys
// further apart, up to kSpreadKeys, and values up to kSpreadValues, are all made larger by what is missing, up to
// 2^6 (keys) or 2^3 (values).  Values stop there because the weights of a step become as much smaller, and smaller
// again by what a token that counts is smaller than one that does not: from 2^6 to 2^-5 at the most, where what float16
// cuts off a weight is 2^-20 of the largest.
constexpr int kSpread = 5, kSpreadKeys = 11, kSpreadValues = 8;
__device__ __forceinline__ int size_of(uint32_t p) {
  const float s = scale_of(p), o = offset_of(p), top = fmaxf(fabsf(o), fabsf(fmaf(15.0f, s, o)));
  return finite_row(p) ? min((int)(__float_as_uint(top) >> 23), 254) : 0;
}

// Half of token t's row, unpacked into its place among the tensor cores' rows, times 2^shift.
template <int D, bool FULL>
__device__ __forceinline__ void spread_row(const uint4 (&codes)[D / 64], uint32_t p, int shift, uint8_t* dst, int t,
                                           int part_of_row) {
  const float scale = scaled(scale_of(p), shift);
  const __half2 low = __float2half2_rn(scale * (FULL ? 262144.0f : 16777216.0f)), high = __float2half2_rn(scale * 1048576.0f),
                o = __float2half2_rn(scaled(offset_of(p), shift));
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    const uint32_t w[4] = {codes[c].x, codes[c].y, codes[c].z, codes[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int chunk = (part_of_row * (D / 64) + c) * 4 + k;
      *reinterpret_cast<uint4*>(dst + (chunk >> 3) * Plan<D>::BLOCK + t * 128 + (((chunk & 7) ^ (t & 7)) << 4)) =
          unpack8<FULL>(w[k], low, high, o);
    }
  }
}

// A row of queries: its running maximum m, its sum l of 2^(x - m), and d: weights are 2^(x - m - d) over the
// step's power of two.
struct Softmax {
  float m = -INFINITY, l = 0.0f, d = 0.0f;

  // m and d after the row's largest score and, as largest(m), its largest product against the new m.  O at o_at
  // follows d; `done` says when it is at rest (null: nothing is there yet).
  template <int D, typename Largest>
  __device__ __forceinline__ void follow(float top, Largest largest, uint32_t o_at, uint64_t* done, uint32_t parity,
                                         int tries, volatile int* stalled) {
    const bool moves = top > m + kSlack;
    const float next = moves ? top : m;
    const float d_here = moves ? d - (next - m) : d;  // the same weights against the new maximum
    const float size = largest(next);
    l *= m == -INFINITY ? 1.0f : ex2(m - next);
    m = next;
    // whole, so that the weight of a token that outdoes all others is exact
    d = size > d_here + kRoom ? ceilf(size) - (kRoom - kSlack) : ceilf(d_here);
    if (done && __any_sync(0xffffffffu, d != d_here)) {
      bar_wait(done, parity, tries, stalled);
      __syncwarp();
      fence_after();
      const float keep = d != d_here ? ex2(d_here - d) : 1.0f;
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        uint32_t y[16];
        load16(y, o_at + c);
        loaded();
        hold(y);
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * keep);
        store16(y, o_at + c);
      }
    }
  }
};

// Half of a step token by token: each key has its own power of two and each value its own (`own`: value's << 16 |
// key's), or, without `own`, scores are `factor` times the products and the values' power is the step's, `now`.  Such
// steps are few, so the scores at `at` are read again for each use, 16 at a time.  A function of its own: within
// the loop over the half steps this code made the others slower (the chunk below 168 us, 165 with the call).
template <int D>
__device__ __noinline__ Softmax by_token(Softmax s, float factor, float now, const uint32_t* own, uint32_t visible0, uint32_t visible1,
                                          uint32_t at, uint32_t o_at, uint64_t* done, uint32_t parity, int tries,
                                          volatile int* stalled) {
  auto read = [&](int c, float (&v)[16], float (&shift)[16]) {
    uint32_t y[16];
    load16(y, at + c);
    loaded();
    hold(y);
    const uint32_t in = (c & 32 ? visible1 : visible0) >> (c & 16);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int both = own ? own[c + k] : 0, undo = -(int)(int16_t)both;
      shift[k] = own ? (float)(both >> 16) : now;
      v[k] = in >> k & 1 ? __uint_as_float(y[k]) * pow2(undo >> 1) * factor * pow2(undo - (undo >> 1)) : -INFINITY;
    }
  };
  float v[16], shift[16], top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 16) {
    read(c, v, shift);
#pragma unroll
    for (int k = 0; k < 16; ++k) top = fmaxf(top, v[k]);
  }
  s.follow<D>(top, [&](float next) {
    float size = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kHalf; c += 16) {
      read(c, v, shift);
#pragma unroll
      for (int k = 0; k < 16; ++k) size = fmaxf(size, v[k] - next - shift[k]);
    }
    return size;
  }, o_at, done, parity, tries, stalled);
  const float m = s.m == -INFINITY ? 0.0f : s.m;
#pragma unroll 1
  for (int c = 0; c < kHalf; c += 16) {  // the weights of 16 tokens lie where scores of no later ones are
    read(c, v, shift);
    uint32_t p[8];
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      s.l += ex2(v[k] - m) + ex2(v[k + 1] - m);
      p[k / 2] = Half2<__half>::pack(ex2(v[k] - m - (s.d + shift[k])), ex2(v[k + 1] - m - (s.d + shift[k + 1])));
    }
    store8(p, at + c / 2);
  }
  return s;
}

// A block's piece of work: the rows of a row tile (or two) and head, and the steps of tokens it takes.
struct Work {
  Sequence seq;
  int b, head, row0, rows;
  int ahead;                 // query i sees ahead + i tokens
  int step0, steps, halves;  // first step of 128 tokens, steps, half steps; no steps: nothing is seen
  int part, parts, tile_head;
  bool some;  // false: this number has no work (in the queue: there is no more)
};
constexpr int kQueue = 8;  // pieces from the one that leaves to the one that is looked up: these are a few steps apart

// Number `n` of the work, found by a whole warp.  The later tiles of a sequence, which see more, come
// first.
template <int RT>
__device__ __forceinline__ Work work_at(const AttendArgs& a, const Split& split, int n, int lane) {
  Work w{};
  const int heads = a.pool.kv_heads;
  w.tile_head = n / split.splits;
  w.part = n - w.tile_head * split.splits;
  const int item = a.kv_heads.div(w.tile_head);
  w.head = w.tile_head - item * heads;
  int before = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < (int)a.batch && !w.some; b0 += 32) {
    Sequence s{0, 0, 0, true};
    int tiles = 0;
    if (b0 + lane < a.batch) {
      s = sequence(a, b0 + lane, false);
      tiles = (s.count * (int)a.group.d + RT - 1) / RT;
    }
    int x = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const uint32_t here = __ballot_sync(0xffffffffu, item >= before + x - tiles && item < before + x);
    if (here) {
      const int from = __ffs(here) - 1;
      w.some = true;
      w.b = b0 + from;
      w.seq.length = __shfl_sync(0xffffffffu, s.length, from);
      w.seq.start = __shfl_sync(0xffffffffu, s.start, from);
      w.seq.count = __shfl_sync(0xffffffffu, s.count, from);
      w.row0 = (before + __shfl_sync(0xffffffffu, x, from) - 1 - item) * RT;
    }
    before = min(before + __shfl_sync(0xffffffffu, x, 31), 0x40000000);
  }
  if (!w.some) return w;
  w.rows = min(RT, w.seq.count * (int)a.group.d - w.row0);
  w.ahead = w.seq.length - w.seq.count + 1;
  const int end = a.causal ? max(0, min(w.seq.length, w.ahead + a.group.div(w.row0 + w.rows - 1))) : w.seq.length;
  const int all = (end + kTile - 1) / kTile;
  const int share = max(kLeastSteps, (all + split.splits - 1) / split.splits);
  w.parts = max(1, (all + share - 1) / share);
  w.some = w.part < w.parts;
  w.step0 = w.part * share;
  w.steps = min(share, all - w.step0);
  w.halves = min(2 * w.steps, (end + kHalf - 1) / kHalf - 2 * w.step0);
  return w;
}

// SPLIT: blocks share row tiles, one piece of work for each block.
template <int D, typename T, bool SPLIT>
__global__ void __launch_bounds__(Plan<D>::WARPS * 32, 1) attend_prompt_kernel(const AttendArgs a, const Split split, const int work) {
  using P = Plan<D>;
  constexpr int TILES = P::TILES, STAGES = P::STAGES, RT = kTile * TILES;
  constexpr int kUnpack = P::UNPACK, kIssue = P::ISSUE;  // first warps of their kind
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t q_full, q_empty, k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES],
      s_full[TILES][2], p_full[TILES][2], o_done[TILES], o_full, w_next, w_full[kQueue],
      w_empty[kQueue];
  __shared__ uint32_t tensor_base;
  __shared__ int stalled_, sh_last, sh_skipped;
  __shared__ int owed_at, owed;  // SPLIT: the count at which this block is expected, and by how many; 0 when it was there
  __shared__ Info infos[kInfos];
  __shared__ Work queue[kQueue];
  __shared__ float factors[2][RT];  // of two pieces' rows
  __shared__ __align__(16) uint32_t range_k[2][4], range_v[2][4];  // of 32 tokens: largest size << 16 | smallest
  __shared__ __align__(16) uint32_t own_shifts[kInfos][kTile];     // of a wide step's tokens: value's << 16 | key's
  volatile int* stalled = &stalled_;
  uint8_t* smem = raw + ((1024 - (smem_of(raw) & 1023)) & 1023);
  // the same in all of a warp's threads, which the compiler sees by the shuffle
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int heads = a.pool.kv_heads;

  if (threadIdx.x == 0) {
    stalled_ = sh_skipped = sh_last = owed = 0;
    bar_init(&q_full, RT);
    bar_init(&q_empty, 1);
    for (int i = 0; i < STAGES; ++i) {
      bar_init(&k_full[i], 2 * kTile);
      bar_init(&v_full[i], 2 * kTile);
      bar_init(&k_empty[i], 1);
      bar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < TILES; ++i) {
      for (int h = 0; h < 2; ++h) {
        bar_init(&s_full[i][h], 1);
        bar_init(&p_full[i][h], kTile);
      }
      bar_init(&o_done[i], 1);
    }
    bar_init(&o_full, 1);
    bar_init(&w_next, 1);
    for (int i = 0; i < kQueue; ++i) {
      bar_init(&w_full[i], 1);
      bar_init(&w_empty[i], 4 * TILES + 8 + 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (blockIdx.x == 0)  // what is wrong with lengths and starts is reported once
    for (int64_t b = threadIdx.x; b < a.batch; b += P::WARPS * 32)
      if (!sequence(a, b, true).ok) sh_skipped = 1;
  // A group's next piece of work, and its return once it is read by the whole warp.
  auto take = [&](int number) -> const Work& {
    bar_wait(&w_full[number % kQueue], number / kQueue & 1, a.wait_limit, stalled);
    __syncwarp();
    return queue[number % kQueue];
  };
  auto give_back = [&](int number) {
    __syncwarp();
    if (lane == 0) bar_arrive(&w_empty[number % kQueue]);
  };
  // All groups begin with this: the scheduling warp must not wait for one that waits for work.
  auto tensor_memory = [&]() {
    fence_before();
    __syncthreads();
    fence_after();
    return tensor_base;
  };

  if (warp < kUnpack) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::SOFTMAX_REGS));
    // ---------------------------------------------------------------- softmax: a row of a tile
    const int tile = warp >> 2, r = threadIdx.x & (kTile - 1), row = tile * kTile + r;
    const uint32_t tensor = tensor_memory();
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 rows of tensor memory
    const uint32_t s_at = tensor + lanes + tile * P::S_COLUMNS, o_at = tensor + lanes + P::O + tile * D;
    uint32_t done0 = 0, done1 = 0, items = 0, steps_done = 0;  // half steps in each place, pieces, steps before this piece
    int number = 0;
#pragma unroll 1
    for (;; ++number) {
      const Work& k = take(number);  // read again where it is used: registers are dear here
      const bool none = !k.some || *stalled;
      if (SPLIT ? any_of<2, RT>(none) : __any_sync(0xffffffffu, none) != 0) break;  // SPLIT: they all meet at the join
      const int seen = row >= k.rows ? 0 : (a.causal ? min(k.seq.length, k.ahead + a.group.div(k.row0 + row)) : k.seq.length);
      const int halves = tile * kTile < k.rows ? k.halves : 0;  // a tile without rows has nothing to wait for
      int left_all = seen - k.step0 * kTile;  // tokens of what is still to come that the row sees
      int least_left = __reduce_min_sync(0xffffffffu, left_all);  // that each of the warp's rows sees
      Softmax softmax;
      float &m = softmax.m, &l = softmax.l, &d = softmax.d;
      bool poisoned = false, far = false;  // far: some |m| of the warp is over kFar
      uint32_t x[2][32];
      auto scores_of = [&](int n) {  // half step n's are there
        bar_wait(&s_full[tile][n & 1], ((n & 1 ? done1 : done0) + (n >> 1)) & 1, a.wait_limit, stalled);
        __syncwarp();
        fence_after();
      };
      // scores are `factor` and the step's factor times the product, in powers of two
      float factor = 0.0f;
      if (halves > 0) {
        scores_of(0);
        factor = factors[items & 1][row];
        load32(x[0], s_at);
        load32(x[1], s_at + 32);
      }
#pragma unroll 1
      for (int n = 0; n < halves; ++n) {
        const int j = n >> 1, h = n & 1;
        const uint32_t at = s_at + h * kHalf, at_next = s_at + (h ^ 1) * kHalf;
        const Info& info = infos[(steps_done + j) & (kInfos - 1)];
        const uint4 head = *reinterpret_cast<const uint4*>(&info);
        const float f = factor * __uint_as_float(head.x) * __uint_as_float(head.y), now = __uint_as_float(head.z);
        const bool special = (head.w >> (16 * h) & 0xffff) != 0, wide = (head.w & 2) != 0;
        const int left = left_all;  // tokens of this half step that the row sees
        const bool masked = least_left < kHalf || special || far;
        left_all -= kHalf;
        least_left -= kHalf;
        loaded();
        hold(x[0]);
        hold(x[1]);
        auto token_by_token = [&](uint32_t visible0, uint32_t visible1) {
          const uint32_t* const own = wide ? own_shifts[(steps_done + j) & (kInfos - 1)] + h * kHalf : nullptr;
          softmax = by_token<D>(softmax, wide ? factor : f, now, own, visible0, visible1, at, o_at,
                                n > 0 ? &o_done[tile] : nullptr, (done0 + done1 + n - 1) & 1, a.wait_limit, stalled);
          far = __any_sync(0xffffffffu, m != -INFINITY && fabsf(m) > kFar);
          stored();
          fence_before();
          bar_arrive(&p_full[tile][h]);
          if (n + 1 < halves) {
            scores_of(n + 1);
            load32(x[0], at_next);
            load32(x[1], at_next + 32);
          }
        };
        uint32_t visible[2] = {0xffffffffu, 0xffffffffu};
        if (masked) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int some = left - w * 32;
            visible[w] = some >= 32 ? 0xffffffffu : (some <= 0 ? 0u : (1u << some) - 1);
            if (special) {
              visible[w] &= ~info.hidden[2 * h + w];
              poisoned |= (visible[w] & info.bad[2 * h + w]) != 0;
            }
          }
          if (wide || far) {
            token_by_token(visible[0], visible[1]);
            continue;
          }
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (masked) {
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              tops[k & 3] = visible[w] >> k & 1 ? fmaxf(tops[k & 3], __uint_as_float(x[w][k])) : tops[k & 3];
        } else {
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int k = 0; k < 32; k += 2)
              tops[k / 2 & 3] = fmaxf(fmaxf(__uint_as_float(x[w][k]), __uint_as_float(x[w][k + 1])), tops[k / 2 & 3]);
        }
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        top = top == -INFINITY ? top : top * f;
        if (__any_sync(0xffffffffu, top > m + fminf(kSlack, d + now + kRoom))) {
          softmax.follow<D>(top, [&](float next) { return top - next - now; }, o_at, n > 0 ? &o_done[tile] : nullptr,
                            (done0 + done1 + n - 1) & 1, a.wait_limit, stalled);
          if (__any_sync(0xffffffffu, m != -INFINITY && fabsf(m) > kFar)) {
            token_by_token(visible[0], visible[1]);
            continue;
          }
        }
        // Weights 2^(x - m - over); `over` stops at 60, where they are under 2^-52 (zeros in float16: values that
        // are tiny beside the others'), so that the softmax's sum, which comes from them, stays in float's range.
        const float over = fminf(d + now, 60.0f);
        const float base = m + over;  // a row that has seen nothing yet: all of its weights are masked
        float2 sum = make_float2(0.0f, 0.0f);
        // Weights of 32 tokens, put over the scores; two at a time where the hardware has it.  The next
        // scores take the registers of those that are done, so that they come while others are worked on.
        auto weigh = [&](auto masked_) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float2 e = fma2(make_float2(__uint_as_float(x[w][2 * k]), __uint_as_float(x[w][2 * k + 1])),
                              make_float2(f, f), make_float2(-base, -base));
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              if constexpr (decltype(masked_)::value) {
                e.x = visible[w] >> (2 * k) & 1 ? e.x : 0.0f;
                e.y = visible[w] >> (2 * k + 1) & 1 ? e.y : 0.0f;
              }
              sum = add2(sum, e);
              p[k] = Half2<__half>::pack(e.x, e.y);
            }
            store16(p, at + w * 16);
            if (n + 1 < halves) {
              if (w == 0) scores_of(n + 1);
              load32(x[w], at_next + w * 32);
            }
          }
        };
        if (masked) weigh(std::true_type{});
        else weigh(std::false_type{});
        l = fmaf(sum.x + sum.y, ex2(over), l);
        stored();
        fence_before();
        bar_arrive(&p_full[tile][h]);
      }
      // ---- the rows' results
      const bool live = row < k.rows;
      const int i = a.group.div(k.row0 + (live ? row : 0)),
                h = k.head * a.group.d + (k.row0 + (live ? row : 0) - i * a.group.d);
      const int64_t o = (int64_t)(k.seq.start + i) * a.q_heads + h;
      const int tile_head = k.tile_head, part = k.part, parts = SPLIT ? k.parts : 1;
      if (halves > 0) {
        bar_wait(&o_full, items & 1, a.wait_limit, stalled);
        __syncwarp();
        fence_after();
      }
      if (poisoned) l = __int_as_float(0x7fffffff);
      // 8 channels of the row, unpacking's order undone
      auto write8 = [&](int d, const float (&v)[8], float k) {
        uint4 w;
        w.x = Half2<T>::pack(v[0] * k, v[1] * k);
        w.y = Half2<T>::pack(v[2] * k, v[3] * k);
        w.z = Half2<T>::pack(v[4] * k, v[5] * k);
        w.w = Half2<T>::pack(v[6] * k, v[7] * k);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + o * D + d) = w;
      };
      const int64_t mine = (int64_t)tile_head * split.splits + part;
      const float inv_l = l == 0.0f ? 0.0f : (SPLIT && parts > 1 ? 1.0f : 1.0f / l);
      const float back0 = ex2(floorf(0.5f * d)) * inv_l, back1 = ex2(d - floorf(0.5f * d));
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = 0;
        if (halves > 0) {
          load32(x, o_at + c);
          loaded();
          hold(x);
        }
        if (live) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[e] = __uint_as_float(x[8 * g + 2 * e]) * back0;
              v[e + 4] = __uint_as_float(x[8 * g + 2 * e + 1]) * back0;
            }
            if (!SPLIT || parts == 1) {
              write8(c + g * 8, v, back1);
            } else {
              float4* to = split.parts + (mine * (D / 4) + c / 4 + g * 2) * RT + row;
              to[0] = make_float4(v[0] * back1, v[1] * back1, v[2] * back1, v[3] * back1);
              to[RT] = make_float4(v[4] * back1, v[5] * back1, v[6] * back1, v[7] * back1);
            }
          }
        }
      }
      if (SPLIT && parts > 1) {
        split.stats[mine * RT + row] = make_float2(m, l);
        __threadfence();
        asm volatile("bar.sync 2, %0;" ::"n"(RT) : "memory");
        if (threadIdx.x == 0) {
          sh_last = arrive(split.arrivals + tile_head, parts);
          owed = 0;
        }
        asm volatile("bar.sync 2, %0;" ::"n"(RT) : "memory");
        if (sh_last) {
          __threadfence();
          const int64_t first = (int64_t)tile_head * split.splits;
          m = -INFINITY;
          for (int p = 0; p < parts; ++p) m = fmaxf(m, __ldcg(&split.stats[(first + p) * RT + row]).x);
          const float base = m == -INFINITY ? 0.0f : m;
          l = 0.0f;
          for (int p = 0; p < parts; ++p) {
            const float2 st = __ldcg(&split.stats[(first + p) * RT + row]);
            l += ex2(st.x - base) * st.y;
          }
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
          for (int d = 0; live && d < D; d += 16) {
            float v[2][8] = {};
            for (int p = 0; p < parts; ++p) {
              const float w = ex2(__ldcg(&split.stats[(first + p) * RT + row]).x - base);
              const float4* from = split.parts + ((first + p) * (D / 4) + d / 4) * RT + row;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 x = __ldcg(from + e * RT);
                v[e >> 1][(e & 1) * 4] += w * x.x;
                v[e >> 1][(e & 1) * 4 + 1] += w * x.y;
                v[e >> 1][(e & 1) * 4 + 2] += w * x.z;
                v[e >> 1][(e & 1) * 4 + 3] += w * x.w;
              }
            }
            write8(d, v[0], inv);
            write8(d + 8, v[1], inv);
          }
        }
      }
      if (live && a.lse && (parts == 1 || sh_last))
        a.lse[o] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
      done0 += (halves + 1) >> 1;
      done1 += halves >> 1;
      if (k.halves > 0) {
        steps_done += k.steps;
        ++items;
      }
      fence_before();
      if (SPLIT) break;
      give_back(number);
    }
  } else if (warp < kIssue) {
    if constexpr (P::UNPACK_REGS > P::LAUNCH_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::UNPACK_REGS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::UNPACK_REGS));
    // ---------------------------------------------------------------- unpacking: half a token's row
    constexpr int CODES = D / 64;  // 16 bytes each of a thread's keys or values
    const int quarter = (warp - kUnpack) & 3, t = quarter * 32 + lane, part_of_row = (warp - kUnpack) >> 2;
    const int64_t side_rows = (int64_t)heads * a.pool.page_size;
    uint4 kc[CODES], vc[CODES];
    uint32_t kp = 0, vp = 0;
    int state = 0;  // 0: past the end, 1: a row of the cache, 2: hidden
    // The step whose pages are looked up (two ahead of the one that is unpacked), and what is known of
    // the one before it.
    int number = 0, slot = 0, slot_now = 0, items = 0, steps_left = 0, token = 0, length = 0, page = -1, place = 0, in_head = 0;
    const int32_t* table = nullptr;
    bool in = false, first = false, valid = true, begun = false;
    auto look_up = [&]() {
      first = steps_left <= 0;
      if (valid && first) {
        do {  // pieces in which nothing is seen are passed over
          const Work& k = take(number);
          valid = !__any_sync(0xffffffffu, !k.some || *stalled);
          steps_left = k.steps;
          length = k.seq.length;
          in_head = k.head;
          token = k.step0 * kTile + t;
          table = a.pages + (int64_t)k.b * a.max_pages;
          if (threadIdx.x == kUnpack * 32) bar_arrive(&w_next);  // time to find the one after it
          if (valid && steps_left <= 0) give_back(number);
          ++number;
        } while (valid && steps_left <= 0);
        slot = number - 1;
      }
      if (!valid) return;
      const int at = a.page_size.div(token);
      in = token < length;
      place = token - at * a.pool.page_size;
      page = in ? __ldg(table + at) : -1;
      token += kTile;
      --steps_left;
    };
    const uint8_t* from = nullptr;
    auto fetch_keys = [&]() {  // of the looked up step, and both rows' parameters
      state = 0;
      kp = vp = 0;
      if (valid && in) {
        if ((unsigned)page < (unsigned)a.pool.num_pages) {
          state = 1;
          const int64_t at = a.pool.row(page, 0, in_head) + place;
          kp = __ldg(a.pool.params + at);
          vp = __ldg(a.pool.params + at + side_rows);
          from = a.pool.codes + at * (D / 2) + part_of_row * (D / 4);
#pragma unroll
          for (int c = 0; c < CODES; ++c) kc[c] = __ldg(reinterpret_cast<const uint4*>(from) + c);
        } else {
          state = 2;
          if (part_of_row == 0) flag(a.status, TANS_DEV_BAD_INDEX);
        }
      }
      if (state != 1) {
#pragma unroll
        for (int c = 0; c < CODES; ++c) kc[c] = make_uint4(0, 0, 0, 0);
      }
    };
    auto fetch_values = [&]() {
      if (state == 1) {
        const uint4* src = reinterpret_cast<const uint4*>(from + side_rows * (D / 2));
#pragma unroll
        for (int c = 0; c < CODES; ++c) vc[c] = __ldg(src + c);
      } else {
#pragma unroll
        for (int c = 0; c < CODES; ++c) vc[c] = make_uint4(0, 0, 0, 0);
      }
    };
    auto spread = [&](bool full, const uint4 (&codes)[CODES], uint32_t p, int shift, uint8_t* dst) {
      if (full) spread_row<D, true>(codes, p, shift, dst, t, part_of_row);
      else spread_row<D, false>(codes, p, shift, dst, t, part_of_row);
    };
    // The queries of the piece whose first step is looked up.  A warp copies 32 rows as they are into
    // their places, LANES lanes a row; then each thread brings a row to float16 by its own power of two.
    auto copy_queries = [&](const Work& k) {
      constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;
      const int row = part_of_row * kTile + t;
      if (row >= RT) return;
      uint8_t* const q_tile = smem + P::Q + part_of_row * P::ROWS;
      const int gr = k.row0 + (row < k.rows ? row : 0), i = a.group.div(gr), h = k.head * a.group.d + (gr - i * a.group.d);
      const T* row_at = static_cast<const T*>(a.q) + (int64_t)(k.seq.start + i) * a.q_ts + h * a.q_hs;
      const int c = lane % LANES;
#pragma unroll 2
      for (int n = lane / LANES; n < 32; n += AT_ONCE) {
        const T* src = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(row_at), n)) + c * 8;
        const bool there = row - lane + n < k.rows;
        const int rr = quarter * 32 + n;
        uint8_t* dst = q_tile + (c >> 3) * P::BLOCK + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
        if (a.vec) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_of(dst)), "l"(src), "r"(there ? 16 : 0)
                       : "memory");
        } else {
          const uint16_t* u = reinterpret_cast<const uint16_t*>(src);
#pragma unroll 1
          for (int e = 0; e < 8; ++e) reinterpret_cast<uint16_t*>(dst)[e] = there ? u[e] : (uint16_t)0;
        }
      }
    };
    auto turn_queries = [&](int item) {
      const int row = part_of_row * kTile + t;
      if (row >= RT) return;
      uint8_t* const q_row = smem + P::Q + part_of_row * P::ROWS + t * 128;
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      float top = 0.0f;
#pragma unroll 2
      for (int c = 0; c < D / 8; ++c) {
        const uint4 x = *reinterpret_cast<const uint4*>(q_row + (c >> 3) * P::BLOCK + (((c & 7) ^ (t & 7)) << 4));
        const float2 f0 = Half2<T>::unpack(x.x), f1 = Half2<T>::unpack(x.y), f2 = Half2<T>::unpack(x.z),
                     f3 = Half2<T>::unpack(x.w);
        top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(f0.x), fabsf(f0.y)), fmaxf(fabsf(f1.x), fabsf(f1.y))),
                               fmaxf(fmaxf(fabsf(f2.x), fabsf(f2.y)), fmaxf(fabsf(f3.x), fabsf(f3.y)))));
      }
      const int e = 13 - max(-113, min(127, (int)(__float_as_uint(top) >> 23) - 127));
      const float up = a.scale_log2 < 0.0f ? -pow2(e) : pow2(e);
      factors[item & 1][row] = fabsf(a.scale_log2) * pow2(-e);
#pragma unroll 2
      for (int c = 0; c < D / 8; ++c) {
        uint4* at = reinterpret_cast<uint4*>(q_row + (c >> 3) * P::BLOCK + (((c & 7) ^ (t & 7)) << 4));
        const uint4 x = *at;
        const float2 f0 = Half2<T>::unpack(x.x), f1 = Half2<T>::unpack(x.y), f2 = Half2<T>::unpack(x.z),
                     f3 = Half2<T>::unpack(x.w);
        uint4 w;  // channels in the order that codes unpack in
        w.x = Half2<__half>::pack(f0.x * up, f2.x * up);
        w.y = Half2<__half>::pack(f0.y * up, f2.y * up);
        w.z = Half2<__half>::pack(f1.x * up, f3.x * up);
        w.w = Half2<__half>::pack(f1.y * up, f3.y * up);
        *at = w;
      }
      fence_smem();
      bar_arrive(&q_full);
    };
    tensor_memory();
    look_up();
    fetch_keys();
    fetch_values();
    begun = first;
    slot_now = slot;
    bool there = valid;
    look_up();
    int stage = 0;
    uint32_t filled = 0;
#pragma unroll 1
    for (uint32_t j = 0;; ++j) {
      if (there && begun) {
        if (items > 0) bar_wait(&q_empty, (items - 1) & 1, a.wait_limit, stalled);
        __syncwarp();
        copy_queries(queue[slot_now % kQueue]);
        give_back(slot_now);
        turn_queries(items);
        ++items;
      }
      // the largest key and value, over the step, and the smallest of those that are not zero
      const int key_size = size_of(kp), value_size = size_of(vp);
      const int most_k = __reduce_max_sync(0xffffffffu, key_size), most_v = __reduce_max_sync(0xffffffffu, value_size),
                least_k = __reduce_min_sync(0xffffffffu, key_size ? key_size : 255),
                least_v = __reduce_min_sync(0xffffffffu, value_size ? value_size : 255);
      if (lane == 0 && part_of_row == 0) {
        range_k[j & 1][quarter] = most_k << 16 | least_k;
        range_v[j & 1][quarter] = most_v << 16 | least_v;
      }
      const bool bad = state == 1 && !finite_row(vp);
      const uint32_t hidden = __ballot_sync(0xffffffffu, state == 2), wrong = __ballot_sync(0xffffffffu, bad);
      if (any_of<1, 256>(!there || *stalled)) break;  // the ranges are there; or some warp has no more
      int key_top = 0, value_top = 0, key_low = 255, value_low = 255;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        key_top = max(key_top, (int)(range_k[j & 1][w] >> 16));
        key_low = min(key_low, (int)(range_k[j & 1][w] & 0xffff));
        value_top = max(value_top, (int)(range_v[j & 1][w] >> 16));
        value_low = min(value_low, (int)(range_v[j & 1][w] & 0xffff));
      }
      const bool wide = key_low + kSpreadKeys < key_top || value_low + kSpreadValues < value_top;
      // what rows are too far apart for the ordinary conversion
      const int more_k = wide ? 0 : max(0, key_top - key_low - kSpread), more_v = wide ? 0 : max(0, value_top - value_low - kSpread);
      const bool full_k = more_k > 0, full_v = more_v > 0;
      const int key_shift = min(kReach + more_k - (wide ? key_size : key_top), kMostShift),
                value_shift = min(kReach + more_v - (wide ? value_size : value_top), kMostShift);
      bar_wait(&k_empty[stage], filled ^ 1, a.wait_limit, stalled);
      Info& info = infos[j & (kInfos - 1)];
      if (lane == 0 && part_of_row == 0) {
        const int undo = -key_shift;  // the same in all, unless the step is wide
        info.key0 = pow2(undo >> 1);
        info.key1 = pow2(undo - (undo >> 1));
        info.value_shift = (float)value_shift;
        info.special[quarter] = ((hidden | wrong) != 0) | (wide ? 2 : 0);
        info.hidden[quarter] = hidden;
        info.bad[quarter] = wrong;
      }
      if (wide && part_of_row == 0)
        own_shifts[j & (kInfos - 1)][t] = (uint32_t)value_shift << 16 | (uint32_t)(key_shift & 0xffff);
      spread(full_k, kc, kp, key_shift, smem + P::K + stage * P::ROWS);
      fence_smem();
      bar_arrive(&k_full[stage]);
      const uint32_t value_params = bad ? 0 : vp;  // a value that is not finite is left to its rows
      fetch_keys();
      begun = first;
      slot_now = slot;
      there = valid;
      look_up();
      bar_wait(&v_empty[stage], filled ^ 1, a.wait_limit, stalled);
      spread(full_v, vc, value_params, value_shift, smem + P::V + stage * P::ROWS);
      fence_smem();
      bar_arrive(&v_full[stage]);
      fetch_values();
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      filled ^= stage == 0;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::ISSUE_REGS));
    if (warp == kIssue) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_of(&tensor_base))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    const uint32_t tensor = tensor_memory();
    if (warp == kIssue) {
      // ---------------------------------------------------------------- products
      // The whole warp walks along, so that operands stay in uniform registers; one thread issues.
      const uint32_t base = smem_of(smem), into = __shfl_sync(0xffffffffu, tensor, 0);
      constexpr uint32_t id_s = instruction(kHalf, false), id_o = instruction(D, true);
      constexpr int HALF = kHalf * 128 >> 4, STAGE = P::ROWS >> 4;  // of an operand's address
      const uint64_t q_at = operand(base + P::Q, 16), k_at = operand(base + P::K, 16),
                     v_at = operand(base + P::V, P::BLOCK);
      const bool one = elected();
      auto scores = [&](int tile, int stage, int h) {
        const uint64_t q = q_at + tile * STAGE, k = k_at + stage * STAGE + h * HALF;
        if (one) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const int in = ((i >> 2) * P::BLOCK + (i & 3) * 32) >> 4;
            mma_ss(into + tile * P::S_COLUMNS + h * kHalf, q + in, k + in, id_s, i > 0);
          }
          commit(&s_full[tile][h]);
        }
        __syncwarp();
      };
      auto values = [&](int tile, int stage, int h, bool more) {
        const uint64_t v = v_at + stage * STAGE + h * HALF;
        if (one) {
#pragma unroll
          for (int i = 0; i < kHalf / 16; ++i)
            mma_ts(into + P::O + tile * D, into + tile * P::S_COLUMNS + h * kHalf + i * 8, v + i * (2048 >> 4), id_o,
                   more || i > 0);
          commit(&o_done[tile]);
        }
        __syncwarp();
      };
      int stage = 0;
      uint32_t filled = 0, items = 0, done0[TILES] = {}, done1[TILES] = {};
#pragma unroll 1
      for (int number = 0;; ++number) {
        const Work& k = take(number);
        const int steps = k.steps, halves = k.halves, tiles = (k.rows + kTile - 1) / kTile;
        const bool some = !__any_sync(0xffffffffu, !k.some || *stalled);
        give_back(number);
        if (!some) break;
        if (steps <= 0) continue;
        bar_wait(&q_full, items & 1, a.wait_limit, stalled);
        bar_wait(&k_full[stage], filled, a.wait_limit, stalled);
        fence_after();
#pragma unroll 1
        for (int n = 0; n < min(2, halves); ++n)
#pragma unroll
          for (int tile = 0; tile < TILES; ++tile)
            if (tile < tiles) scores(tile, stage, n);
        if (one) {
          commit(&k_empty[stage]);
          if (halves <= 2) commit(&q_empty);
        }
        __syncwarp();
#pragma unroll 1
        for (int n = 0; n < halves; ++n) {
          const int h = n & 1, next = stage + 1 == STAGES ? 0 : stage + 1;
          const uint32_t next_filled = filled ^ (next == 0);
          if (h == 0) bar_wait(&v_full[stage], filled, a.wait_limit, stalled);
#pragma unroll
          for (int tile = 0; tile < TILES; ++tile) {
            if (tile >= tiles) continue;
            bar_wait(&p_full[tile][h], ((h ? done1[tile] : done0[tile]) + (n >> 1)) & 1, a.wait_limit, stalled);
            fence_after();
            values(tile, stage, h, n > 0);
            if (n + 2 < halves) {
              if (h == 0 && tile == 0) {
                bar_wait(&k_full[next], next_filled, a.wait_limit, stalled);
                fence_after();
              }
              scores(tile, next, h);
            }
          }
          if (one && n + 3 == halves) commit(&q_empty);  // no product reads these queries any more
          __syncwarp();
          if (h == 1 || n + 1 == halves) {  // the step's last half
            if (one) {
              commit(&v_empty[stage]);
              if ((n >> 1) + 1 < steps) commit(&k_empty[next]);
            }
            __syncwarp();
            stage = next;
            filled = next_filled;
          }
        }
        if (one) commit(&o_full);
        __syncwarp();
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile) {
          if (tile >= tiles) continue;
          done0[tile] += (halves + 1) >> 1;
          done1[tile] += halves >> 1;
        }
        ++items;
      }
      // nothing is in flight when the tensor memory is given back, even after a wait that ran out
      volatile int late = 0;
      if (items > 0) bar_wait(&o_full, (items - 1) & 1, kTries, &late);
    } else if (warp == kIssue + 1) {
      // ---------------------------------------------------------------- scheduling
      // The first pieces are the blocks' by their numbers, the others whoever's is free: pieces of a
      // causal prompt differ by the tokens that they see, the largest come first.
      int number = 0, n = blockIdx.x, steps = 0;  // of the piece before
#pragma unroll 1
      for (;;) {
        Work w{};
        if (n < work) w = work_at<RT>(a, split, n, lane);
        if (SPLIT && w.some && w.parts > 1 && lane == 0) {
          owed_at = w.tile_head;
          owed = w.parts;
        }
        if (n < work && !w.some) {
          n = SPLIT ? work : gridDim.x + __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(split.arrivals, 1) : 0, 0);
          continue;
        }
        bar_wait(&w_empty[number % kQueue], number / kQueue & 1 ^ 1, a.wait_limit, stalled);
        if (__any_sync(0xffffffffu, *stalled)) break;  // the place may be in use; nobody waits for it
        if (lane == 0) {
          queue[number % kQueue] = w;
          bar_arrive(&w_full[number % kQueue]);
        }
        __syncwarp();
        if (!w.some) break;
        // One that is taken earlier than it is needed may be one that another block would end sooner.  The one
        // before it goes first: 16 tries more for each of its steps, which take two or three microseconds.
        bar_wait(&w_next, number & 1, a.wait_limit + 16 * steps, stalled);
        steps = w.steps;
        ++number;
        n = SPLIT || __any_sync(0xffffffffu, *stalled) ? work : gridDim.x + __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(split.arrivals, 1) : 0, 0);
      }
      // every block has had its last number when the last of them comes here
      if (!SPLIT && lane == 0 && arrive(split.arrivals + 1, gridDim.x)) split.arrivals[0] = 0;
    }
  }
  fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && stalled_) flag(a.status, TANS_DEV_STALLED);
  // A block that stalled before its join arrives all the same: the counts are zero after every call.  (Its row
  // tile may then be joined by nobody, or with what is not valid: the flag says so.)
  if (SPLIT && threadIdx.x == 0 && owed > 0) arrive(split.arrivals + owed_at, owed);
  if (warp == kIssue) {
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tensor_base));
  }
  zero_unowned<T>(a, D, blockIdx.x * (int64_t)(P::WARPS * 32) + threadIdx.x, (int64_t)gridDim.x * P::WARPS * 32);
  if (blockIdx.x == 0 && sh_skipped)
    zero_unanswered(a, D, threadIdx.x, P::WARPS * 32, RT, work / (split.splits * heads));
}

// Row tiles times heads, at most: one tile that is not full for each sequence that has queries.
int64_t most_tiles(int tile, int64_t total_rows, int64_t sequences, int kv_heads) {
  return std::max<int64_t>(1, (total_rows / tile + sequences) * kv_heads);
}

// Blocks for each row tile: all tiles at once when they fill the SMs; else the number that ends first,
// with as many rounds of blocks as it takes and a block's start and end (and its part in the join)
// costing it as much as 4 steps.  The lengths are only known by their bound here; a block that finds
// nothing to do ends at once.
int splits_for(int64_t tiles, int64_t max_tokens) {
  const int sms = sm_count();
  const int64_t steps = (max_tokens + kTile - 1) / kTile;
  if (tiles >= sms) return 1;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int n = 1; n <= 64 && tiles * n <= 2 * sms && (n == 1 || (n - 1) * kLeastSteps < steps); ++n) {
    const int64_t cost = (tiles * n + sms - 1) / sms * ((steps + n - 1) / n + 4);
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

template <int D, typename T>
int launch(const AttendArgs& a, void* workspace, cudaStream_t s) {
  using P = Plan<D>;
  constexpr int RT = kTile * P::TILES;
  const int64_t tiles = most_tiles(RT, a.total_queries * a.group.d, std::min(a.batch, a.total_queries), a.pool.kv_heads);
  if (tiles > 0x3fffffff) return TANS_E_TOO_LARGE;
  Split split{1, nullptr, nullptr, nullptr};
  split.splits = splits_for(tiles, a.max_pages * a.pool.page_size);
  split.arrivals = static_cast<int*>(workspace);
  split.stats = reinterpret_cast<float2*>(static_cast<char*>(workspace) + Join::kArrivalBytes);
  split.parts = reinterpret_cast<float4*>(split.stats + tiles * split.splits * RT);
  const int work = (int)tiles * split.splits;
  auto go = [&](auto split_, int blocks) {
    auto* kernel = &attend_prompt_kernel<D, T, decltype(split_)::value>;
    static std::atomic<bool> ready[64];  // of this kernel, by device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TANS_E_CUDA;
    if (!ready[dev].load(std::memory_order_relaxed)) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::BYTES) != cudaSuccess)
        return TANS_E_CUDA;
      ready[dev].store(true, std::memory_order_relaxed);
    }
    kernel<<<blocks, P::WARPS * 32, P::BYTES, s>>>(a, split, work);
    note_launch();
    return cudaGetLastError() == cudaSuccess ? TANS_OK : TANS_E_CUDA;
  };
  return split.splits > 1 ? go(std::true_type{}, work)
                          : go(std::false_type{}, std::min(work, sm_count()));
}

}  // namespace

size_t attend_prompt_workspace(int head_dim, int64_t total_rows, int64_t sequences, int kv_heads, int64_t max_tokens) {
  const int64_t rows = head_dim == 256 ? kTile : 2 * kTile;
  const int64_t tiles = most_tiles((int)rows, total_rows, sequences, kv_heads);
  const int splits = splits_for(tiles, max_tokens);
  return align_up(Join::kArrivalBytes + (splits == 1 ? 0 : (size_t)tiles * splits * rows * (8 + head_dim * 4)));
}

int launch_attend_prompt(const AttendArgs& a, int dtype, void* workspace, cudaStream_t s) {
  auto by_dim = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return a.pool.head_dim == 64    ? launch<64, T>(a, workspace, s)
           : a.pool.head_dim == 128 ? launch<128, T>(a, workspace, s)
                                    : launch<256, T>(a, workspace, s);
  };
  return dtype == TANS_BF16 ? by_dim(static_cast<__nv_bfloat16*>(nullptr)) : by_dim(static_cast<__half*>(nullptr));
}

}  // namespace kv4
}  // namespace tans
