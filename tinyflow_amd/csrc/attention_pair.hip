// Attention on fp16 pairs: forward_kernel, dq_kernel and dkv_kernel, and pack_kernel, which splits their operands.
//
// A block of 32 rows of an operand (queries, their gradients, keys or values of one head) is multiplied by the power of two that brings its
// largest value into [2^14, 2^15), and each element is made of two fp16 numbers, h its nearest one and l the nearest to what is left: three
// products of the fp16 instruction, h h' + h l' + l h', take the place of one of the fp32 instruction, which has a sixteenth of its rate.  What is
// left off is 2^-23 of an element, or 2^-40 of its block's largest value where that is more, and l l', up to 2^-22 of a product.
// Scales are a block's, so a product's scale is known for a whole tile and costs nothing: it is part of the factor of a score, of the
// exponent of p, of ds.  The sum over blocks has a scale of its own for each row (out, dq) or key (dk, dv): that of the largest p v, ds k, ds q or p do that it
// has had, so that what is left off p or ds is 2^-32 of that at most, whatever lies beside the row or was next to nothing in it.  When a larger one comes the
// sum is multiplied; a lane holds one row's or key's, so that is one factor a lane.
//
// Bound: the part's power and, with one or two waves a SIMD, the vector work between the products.  4 096 causal tokens, 16 heads on 4 of 128, 69 GFLOP
// forward: pack 19 us, forward 178 to 206 (334 to 386 TFLOP/s; the fp32 instruction 1 094); backward: pack 54, dq 277 to 327 (315 to 372, three products), dkv 396 to 470
// (292 to 347, four).  A product of the library on the fp16 instruction reaches a third of 1 178 to 1 347.
//
// A block has kBad for its exponent if it holds an infinity or a NaN, or gradients with a row whose statistic or delta is not finite, if its values pass
// 2^55 or stay below 2^-96, or if a row or a column of it is smaller than 2^-16 of its largest value and would lose its digits (of queries and keys in the forward
// pass only the scores count).  Workgroups that meet one, or blocks of queries and keys so large that what is left off would show in a score
// (Exponents::least_sum), leave their rows to the fp32 kernels.  Rows that see nothing and keys that nothing sees are packed as zeros, whatever they hold.
#include "attention.h"
#include "internal.h"
#include "lanes.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace tf {
namespace attention {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int V>
using IC = std::integral_constant<int, V>;

template <int N, class F, int... I>
__device__ __forceinline__ void static_for_impl(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for_impl<N>(f, std::make_integer_sequence<int, N>{});
}

constexpr int kFragment = 1024;  // bytes: 32 rows x 16 of fp16, a wave's lanes one behind the other
constexpr int kInfoBytes = 1024;  // of a block of rows: eight arrays of 32, see Info
constexpr int kSmallest = 110;   // the largest exponent: of zeros, and of queries and keys that no score notices
constexpr int kLargest = -40;
constexpr int kSpansReadByAll = 2048;
constexpr int kNoUnit = INT32_MAX / 2;  // of a sum of nothing
constexpr int kFirstHeld = 60;

// Bytes of a block of 32 rows: DP columns of h and l.
__host__ __device__ constexpr int64_t block_size(int dp) { return dp * 128; }

// ------------------------------------------------------------------------------ splitting

// By value: a bit cast of an element of a vector takes the vector's first one, whichever it is.
__device__ inline uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }

enum Info { kStat = 0, kDelta, kLo, kHi, kSlope, kNear };

struct Job {
  const float *src;
  bool of_rows;
  bool digits;       // whether every row's and column's own digits count, not only the scores'
  char *plain, *transposed;
  int *exponents;
  int first;         // workgroup
};
struct Pack {
  Job jobs[4];
  int n_jobs, row_blocks, key_blocks;
  int2 *seen;        // of each sequence, the keys between the first and the last that any query sees; null: each workgroup finds out
  // backward, by job 1, the gradients of the output:
  const float *out, *stat;
  Row *rows;         // of all
  float *info;       // [b, key head][block of rows][8][32]
  Hull *hulls;
};

__device__ inline void split(float x, _Float16 &h, _Float16 &l) {
  h = (_Float16)x;
  l = (_Float16)(x - (float)h);
}

// The first key that any of a sequence's queries sees, and the one behind the last, by THREADS threads.
template <int THREADS>
__device__ inline void span_hull(const Call &c, int b, int (&hull)[2]) {
  if (threadIdx.x == 0) hull[0] = c.tk, hull[1] = 0;
  __syncthreads();
  int lo = c.tk, hi = 0;
  for (int i = threadIdx.x; i < c.tq; i += THREADS) {
    int l, h;
    c.seen(b, i, l, h);
    if (l < h) lo = min(lo, l), hi = max(hi, h);
  }
  atomicMin(&hull[0], lo);
  atomicMax(&hull[1], hi);
  __syncthreads();
}
__global__ __launch_bounds__(1024) void seen_kernel(const Call c, int2 *seen) {
  __shared__ int hull[2];
  span_hull<1024>(c, (int)blockIdx.x, hull);
  if (threadIdx.x == 0) seen[blockIdx.x] = make_int2(hull[0], hull[1]);
}

// A workgroup a block; bound by HBM, 5.0 to 5.4 TB/s with long heads.  Plain form: step s of 16 columns, h then l, lane: row lane % 32, columns 16 s + 8 (lane / 32) + 0..7.  Transposed: columns 32 d
// + lane % 32, rows 16 t + key_of's order, so that a tile's probabilities are the other operand as they lie.
template <int DP>
__global__ __launch_bounds__(kThreads) void pack_kernel(const Call c, const Pack p) {
  __shared__ __align__(16) float tile[32][DP + 4];
  __shared__ uint32_t most[32];
  __shared__ int finds[4];
  __shared__ int hull[2];
  int which = 0;
  for (int i = 1; i < p.n_jobs; ++i) which = (int)blockIdx.x >= p.jobs[i].first ? i : which;
  const Job &job = p.jobs[which];
  const int blocks = job.of_rows ? p.row_blocks : p.key_blocks;
  const int at = (int)blockIdx.x - job.first, head = at / blocks, block = at % blocks, b = head / c.key_heads, g = head % c.key_heads;
  const int tid = threadIdx.x, row = tid / 8, n = block * 32 + row;
  bool used;
  Row info = {0.f, 0.f, 0, 0};
  if (job.of_rows) {
    if (n < c.rows) c.seen(b, n / c.group, info.lo, info.hi);
    used = info.lo < info.hi;
  } else {
    // keys that any query sees lie between the first and the last of them
    int lo = 0, hi = c.tk;
    if (c.spans) {
      if (p.seen) {
        lo = p.seen[b].x, hi = p.seen[b].y;
      } else {
        span_hull<kThreads>(c, b, hull);
        lo = hull[0], hi = hull[1];
      }
    }
    used = n < c.tk && n >= lo && n < hi;
  }
  const float *src = job.src + (used ? job.of_rows ? c.query_at(b, g, n) : c.key_at(b, g, n) : 0);
  f32x4 x[DP / 32];
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) {
    const int col = 32 * e + tid % 8 * 4;
    x[e] = used && col < c.dim ? load4(src + col, c.dim - col) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, bits_of(x[e][i]) & 0x7fffffffu);
  }
#pragma unroll
  for (int step = 1; step < 8; step *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, step));
  if (tid % 8 == 0) most[row] = top;
  __syncthreads();
  uint32_t largest = 0, least = 0x7f800000u;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t v = most[i];
    largest = max(largest, v);
    least = v ? min(least, v) : least;
  }
  const int field = (int)(largest >> 23);
  int exponent = min(kSmallest, 141 - field);
  if (largest >= 0x7f800000u || exponent < kLargest) exponent = kBad;
  if (job.digits && largest && ((int)(least >> 23) < field - 16 || 141 - field > kSmallest)) exponent = kBad;
  if (p.info && which == 1) {  // what the backward kernels read of the rows
    __shared__ Row of_rows[32];
    float delta = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) {
      const int col = 32 * e + tid % 8 * 4;
      if (!used || col >= c.dim) continue;
      const f32x4 o = load4(p.out + (src - job.src) + col, c.dim - col);
      delta += (x[e][0] * o[0] + x[e][1] * o[1]) + (x[e][2] * o[2] + x[e][3] * o[3]);
    }
    delta = lanes::sum_over<8>(delta);
    if (tid % 8 == 0) {
      if (used) info.stat = c.taken(b, g, n, info.lo, info.hi, p.stat[c.stat_at(b, g, n)]);
      if (!used || info.stat == kNone) info = Row{0.f, 0.f, 0, 0};
      else info.delta = delta;
      if (n < c.rows) p.rows[(int64_t)head * c.rows + n] = info;
      of_rows[row] = info;
    }
    // A row that has seen an infinity or a NaN has passed it to its statistic or to delta, and 0 times that is no gradient of the keys that it
    // does not see: the fp32 kernels choose by mask.
    if (__syncthreads_or(tid % 8 == 0 && !(finite(info.stat) && finite(info.delta)))) exponent = kBad;
    if (tid < 64) {
      const int r = block * 32 + tid % 32;
      const Row mine = of_rows[tid % 32];
      Hull seen;
      seen.of(mine.lo, mine.hi, true);
      if (seen.lo >= seen.hi) seen.lo = seen.hi = 0;
      // rows that see nothing, or that are none, keep the block from covering anything
      if (__any(mine.lo >= mine.hi)) seen.inner_lo = INT32_MAX, seen.inner_hi = 0;
      const int64_t of_block = (int64_t)head * blocks + block;
      if (tid < 32) {
        float *to = p.info + of_block * (kInfoBytes / 4) + tid;
        to[32 * kStat] = mine.stat;
        to[32 * kDelta] = mine.delta;
        to[32 * kLo] = __builtin_bit_cast(float, mine.lo);
        to[32 * kHi] = __builtin_bit_cast(float, mine.hi);
        to[32 * kSlope] = c.slopes && r < c.rows ? c.slopes[g * c.group + r % c.group] * kLog2e : 0.f;
        to[32 * kNear] = r < c.rows ? (float)c.nearest(c.own(b, r / c.group), mine.lo, mine.hi) : 0.f;
      }
      if (tid == 0) p.hulls[of_block] = seen;
    }
  }
  // Elements smaller than 2^-16 of the largest, zeros among them, of the wave's eight rows.  A column of nothing else has one in each row that is not all zeros;
  // as many beside what is zero by itself, rows and columns that are none, are a reason to look for it.
  const float not_small = __builtin_bit_cast(float, (uint32_t)max(field - 16, 0) << 23);
  int smalls = 0;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (job.digits) smalls += __popcll(__ballot(fabsf(x[e][i]) < not_small));
      x[e][i] = __builtin_ldexpf(x[e][i], exponent);
    }
    *reinterpret_cast<f32x4 *>(&tile[row][32 * e + tid % 8 * 4]) = x[e];
  }
  const int live_rows = __popcll(__ballot(top != 0)) / 8;
  if (tid % 64 == 0) finds[tid / 64] = live_rows > 0 && smalls - 8 * DP + live_rows * c.dim >= live_rows;
  __syncthreads();
  int *const exponent_at = job.exponents + (int64_t)head * blocks + block;
  if (exponent == kBad) {
    if (tid == 0) *exponent_at = kBad;
    return;
  }
  const int64_t to = ((int64_t)head * blocks + block) * block_size(DP);
  if (job.plain)
#pragma unroll
    for (int u = tid; u < DP * 4; u += kThreads) {
      const int r = u % 32, eighth = u / 32;
      f16x8 h, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        _Float16 a, d;
        split(tile[r][8 * eighth + e], a, d);
        h[e] = a;
        l[e] = d;
      }
      char *out = job.plain + to + eighth / 2 * 2 * kFragment + (eighth % 2 * 32 + r) * 16;
      *reinterpret_cast<f16x8 *>(out) = h;
      *reinterpret_cast<f16x8 *>(out + kFragment) = l;
    }
  if (job.transposed)
#pragma unroll
    for (int u = tid; u < DP * 4; u += kThreads) {
      const int col = u % DP, t = u / DP / 2, half = u / DP % 2;
      f16x8 h, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        _Float16 a, d;
        split(tile[16 * t + key_of(e, half)][col], a, d);
        h[e] = a;
        l[e] = d;
      }
      char *out = job.transposed + to + (col / 32 * 2 + t) * 2 * kFragment + (half * 32 + col % 32) * 16;
      *reinterpret_cast<f16x8 *>(out) = h;
      *reinterpret_cast<f16x8 *>(out + kFragment) = l;
    }
  // Columns that are that small in all rows, and not all zeros, cannot be split.  Of a single row they are no column yet: its elements are what they are beside
  // its largest.
  if (finds[0] | finds[1] | finds[2] | finds[3]) {
    const uint64_t rows = __ballot(tid % 64 < 32 && most[tid % 32] != 0);
    float top_of = 0.f;
    if (tid < DP)
#pragma unroll 4
      for (int r = 0; r < 32; ++r) top_of = fmaxf(top_of, fabsf(tile[r][tid]));
    if (__syncthreads_or(top_of > 0.f && top_of < __builtin_ldexpf(not_small, exponent)) && (rows & (rows - 1)) != 0) exponent = kBad;
  }
  if (tid == 0) *exponent_at = exponent;
}

// ------------------------------------------------------------------------------ what the products share

__device__ inline f16x8 fragment(const char *at) { return *reinterpret_cast<const f16x8 *>(at); }
__device__ inline f32x16 mfma(f16x8 a, f16x8 b, f32x16 sum) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, sum, 0, 0, 0); }
__device__ inline f32x16 zeros() {
  f32x16 z;
#pragma unroll
  for (int v = 0; v < 16; ++v) z[v] = 0.f;
  return z;
}

// A wave's operand of 32 rows or keys in the plain form, in registers.
template <int DP>
struct Held {
  f16x8 h[DP / 16], l[DP / 16];
  __device__ inline void load(const char *block) {
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      h[s] = fragment(block + 2 * s * kFragment + lane * 16);
      l[s] = fragment(block + (2 * s + 1) * kFragment + lane * 16);
    }
  }
  // Odd lanes' elements with the other sign.  The instruction cuts a sum that is smaller than its products off downwards: what
  // comes out is 3.3e-8 too small on the average where the sum before was about 0.1 and the 16 products are about 1 each.  In ds such an error is one of every p, which turns all of a head's
  // queries the same way, and over 65 536 rows the gradients of what scales the heads were off by 2.5e-6 of themselves; where every other row, or key, has
  // the opposite error, by 1.2e-6, which is what the fp32 instruction gives.
  __device__ inline void alternate() {
    const uint32_t sign = threadIdx.x % 2 ? 0x80008000u : 0u;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      h[s] = __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, h[s]) ^ sign);
      l[s] = __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, l[s]) ^ sign);
    }
  }
  // Waits for them, before loads that the compiler does not count are under way.  APART: in the registers that only matrix instructions
  // read, where the others are too few for what they are needed for.
  template <bool APART>
  __device__ inline void wait() {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
      if constexpr (APART) asm volatile("" : "+a"(h[s]), "+a"(l[s]));
      else asm volatile("" : "+v"(h[s]), "+v"(l[s]));
  }
};

// Products of blocks that lie one behind the other in LDS, in the plain form, with what the wave holds for each.  The fragments are read READ_AHEAD
// steps before they are multiplied, and `between(n)` is what is computed while the n-th instruction runs, of which a step has three: a wave issues
// in order, so only what stands behind a single matrix instruction, before the next, runs beside it (five vector instructions do in the 34 cycles of
// one; from the eighth on each costs five cycles).  The order is kept as it stands here; left to itself the compiler reads a fragment, waits
// for it and multiplies.
template <int DP, int N, int READ_AHEAD, class Between>
__device__ __forceinline__ void products(const char *blocks, const Held<DP> *const (&held)[N], f32x16 (&sum)[N], const Between &between) {
  constexpr int STEPS = DP / 16, ALL = N * STEPS, AHEAD = READ_AHEAD < ALL ? READ_AHEAD : ALL;
  const char *const at = blocks + threadIdx.x % 64 * 16;
  f16x8 h[ALL], l[ALL];
  auto read = [&](auto n_c) {
    constexpr int n = decltype(n_c)::value;
    h[n] = fragment(at + 2 * n * kFragment);
    l[n] = fragment(at + (2 * n + 1) * kFragment);
  };
  static_for<AHEAD>([&](auto n) { read(n); });
  __builtin_amdgcn_sched_barrier(0);
  static_for<ALL>([&](auto n_c) {
    constexpr int n = decltype(n_c)::value, block = n / STEPS, step = n % STEPS;
    if constexpr (step == 0) sum[block] = zeros();
    if constexpr (n + AHEAD < ALL) read(IC<n + AHEAD>{});
    sum[block] = mfma(l[n], held[block]->h[step], sum[block]);
    between(IC<3 * n>{});
    __builtin_amdgcn_sched_barrier(0);
    sum[block] = mfma(h[n], held[block]->l[step], sum[block]);
    between(IC<3 * n + 1>{});
    __builtin_amdgcn_sched_barrier(0);
    sum[block] = mfma(h[n], held[block]->h[step], sum[block]);
    between(IC<3 * n + 2>{});
    __builtin_amdgcn_sched_barrier(0);
  });
}

// 16 values of a tile as the other operand of a product over its rows: instruction t takes values 8 t .. 8 t + 7.
struct Weights {
  f16x8 h[2], l[2];
  // values 2 n and 2 n + 1
  template <int n>
  __device__ __forceinline__ void set(float a, float b) {
    constexpr int t = n / 4, e = 2 * (n % 4);
    const f32x2 x = {a, b};
    const f16x2 top = __builtin_convertvector(x, f16x2);
    // what is left, from the fp16 number as it lies: the compiler would widen it first
    f32x2 left;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(left[0]) : "v"(top), "v"(a));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(left[1]) : "v"(top), "v"(b));
    const f16x2 rest = __builtin_convertvector(left, f16x2);
    h[t][e] = top[0];
    h[t][e + 1] = top[1];
    l[t][e] = rest[0];
    l[t][e + 1] = rest[1];
  }
};

// sum[d] += of a transposed block, `between` as above.  The weights' second halves may be set in it, before the instruction 3 DP / 32.
template <int DP, int READ_AHEAD, class Between>
__device__ __forceinline__ void add_product(f32x16 (&sum)[DP / 32], const char *block, const Weights &w, const Between &between) {
  constexpr int D = DP / 32, ALL = 2 * D, AHEAD = READ_AHEAD < ALL ? READ_AHEAD : ALL;
  const char *const at = block + threadIdx.x % 64 * 16;
  f16x8 h[ALL], l[ALL];
  auto read = [&](auto n_c) {
    constexpr int n = decltype(n_c)::value, index = n % D * 2 + n / D;
    h[n] = fragment(at + index * 2 * kFragment);
    l[n] = fragment(at + (index * 2 + 1) * kFragment);
  };
  static_for<AHEAD>([&](auto n) { read(n); });
  __builtin_amdgcn_sched_barrier(0);
  static_for<ALL>([&](auto n_c) {
    constexpr int n = decltype(n_c)::value, t = n / D, d = n % D;
    if constexpr (n + AHEAD < ALL) read(IC<n + AHEAD>{});
    sum[d] = mfma(l[n], w.h[t], sum[d]);
    between(IC<3 * n>{});
    __builtin_amdgcn_sched_barrier(0);
    sum[d] = mfma(h[n], w.l[t], sum[d]);
    between(IC<3 * n + 1>{});
    __builtin_amdgcn_sched_barrier(0);
    sum[d] = mfma(h[n], w.h[t], sum[d]);
    between(IC<3 * n + 2>{});
    __builtin_amdgcn_sched_barrier(0);
  });
}
// COUNT pieces of work over the places [FIRST, FIRST + PLACES): do_piece(k) at place n.
template <int n, int FIRST, int PLACES, int COUNT, class F>
__device__ __forceinline__ void spread(const F &do_piece) {
  if constexpr (n >= FIRST && n < FIRST + PLACES)
    static_for<COUNT>([&](auto k_c) {
      if constexpr (decltype(k_c)::value * PLACES / COUNT == n - FIRST) do_piece(k_c);
    });
}
struct Nothing {
  template <class T>
  __device__ __forceinline__ void operator()(T) const {}
};

template <int N>
__device__ inline void multiply(f32x16 (&sum)[N], float by) {
#pragma unroll
  for (int d = 0; d < N; ++d) sum[d] *= by;
}
// Keeps sums in the registers that only matrix instructions work on: where a branch multiplies them, the compiler otherwise holds them in the
// others and moves all of them there and back at every step.
template <bool APART, int N>
__device__ __forceinline__ void keep(f32x16 (&sum)[N]) {
  if constexpr (APART)
#pragma unroll
    for (int d = 0; d < N; ++d) asm volatile("" : "+a"(sum[d]));
}

// Brings one or two KB from `from` + OFFSET to LDS at `to` + OFFSET, 16 bytes a lane.  Written out because the compiler takes every read of LDS for a
// reader of the loads into it that are under way, and waits for them; `arrived` is the wait that they need.  They write no register.
template <int OFFSET, bool TWO>
__device__ __forceinline__ void fetch(uint32_t to, const char *from) {
  const uint32_t lane = threadIdx.x % 64 * 16u;
  if constexpr (TWO)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3\n\tglobal_load_lds_dwordx4 %1, %2 offset:%4" ::"s"(to), "v"(lane),
                 "s"(from), "n"(OFFSET), "n"(OFFSET + 1024)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" ::"s"(to), "v"(lane), "s"(from), "n"(OFFSET) : "memory");
}
// Everything that this wave has fetched, and read from LDS, has arrived, in all waves.
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ inline uint32_t lds_address(const char *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p; }

__device__ inline const char *uniform(const char *p) {
  const uint64_t v = (uint64_t)p;
  return (const char *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}

// What the launch before has written and this one only reads, at an address that the wave shares: by a scalar load, which leaves the count of
// the vector loads under way alone.
__device__ inline int scalar(const int *p) { return *(const __attribute__((address_space(4))) int *)uniform((const char *)p); }
// 2^-(a + b) factor, for scores: not below 2^-120, where a product of less than 2^37 is no score, so that it times the -infinity of a masked one is that
__device__ inline float unscaled(float factor, int a, int b) { return fmaxf(__builtin_ldexpf(factor, -(a + b)), 0x1p-120f); }


// Block `index` of each of N operands, one behind the other in LDS from `to` on: each of four waves fetches a quarter of each.
template <int DP, int N>
struct Blocks {
  static constexpr int QUARTER = DP / 32, EACH = (QUARTER + 1) / 2, kCount = N * EACH;  // fragments, fetches
  const char *from[N];
  uint32_t to;
  __device__ __forceinline__ Blocks(const char *const (&of)[N], int64_t index, uint32_t at) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % 4);
    to = __builtin_amdgcn_readfirstlane(at + (uint32_t)(wave * QUARTER * kFragment));
    static_for<N>([&](auto n) { from[decltype(n)::value] = uniform(of[decltype(n)::value] + index * block_size(DP) + wave * QUARTER * kFragment); });
  }
  template <int f>
  __device__ __forceinline__ void one() const {
    constexpr int n = f / EACH, i = f % EACH * 2;
    fetch<i * kFragment, (i + 1 < QUARTER)>(to + (uint32_t)(n * block_size(DP)), from[n]);
  }
  __device__ __forceinline__ void all() const {
    static_for<kCount>([&](auto f) { one<decltype(f)::value>(); });
  }
};

// ------------------------------------------------------------------------------ forward

// 128 rows a workgroup, of two groups of four waves with 32 rows each: one group takes the even steps of 32 keys, one the odd ones, and the
// second's sums join the first's through LDS at the end.  While a step is worked on the next one is on its way into LDS.  Two waves a SIMD then
// belong to one workgroup, which takes half as long, and a causal pass, whose workgroups differ as the rows do, ends with
// light ones on every CU.  PLAIN: neither cap nor bias.
template <int DP, bool PLAIN>
__global__ __launch_bounds__(2 * kThreads, DP <= 64 ? 4 : 2) void forward_kernel(const Call c, const char *qs, const char *ks, const char *vs, const Exponents ex,
                                                                                 float *out, float *stat, const Pieces pieces, int tiles) {
  constexpr int BLOCK = (int)block_size(DP);
  constexpr int AHEAD = DP <= 64 ? 1 : 3;
  __shared__ __align__(16) char lds[2][2][2 * BLOCK];  // [parity][group]
  __shared__ int room[8][4];
  __shared__ float marks[2][kRows];
  const int heads = c.batch * c.key_heads;
  const int bg = (int)blockIdx.x % heads, rest = (int)blockIdx.x / heads;
  const int b = bg / c.key_heads, g = bg % c.key_heads, tile = tiles - 1 - rest % tiles, piece = rest / tiles;
  const int lane = threadIdx.x % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % 4);
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  const int r = tile * kRows + wave * 32 + lane % 32;
  const bool live = r < c.rows;
  const int i = (live ? r : c.rows - 1) / c.group;
  int lo, hi, at;
  c.seen(b, i, lo, hi, at);
  const int near = c.nearest(at, lo, hi);
  Hull mine;
  mine.of(lo, hi, live);
  const Hull all = mine.all(room);  // the second group's waves have the first's rows
  const int first = all.first(), steps = all.steps();
  if (__syncthreads_or(ex.bad_rows(bg, tile * (kRows / 32), first, steps))) return;
  const int begin = first + (int)((int64_t)steps * piece / pieces.count), end = first + (int)((int64_t)steps * (piece + 1) / pieces.count);
  const int block = min(tile * (kRows / 32) + wave, ex.row_blocks - 1);
  const int64_t row_block = (int64_t)bg * ex.row_blocks + block, key_block = (int64_t)bg * ex.key_blocks;
  const int eq = scalar(ex.q + row_block);
  const float slope = !PLAIN && c.slopes ? c.slopes[g * c.group + (live ? r : 0) % c.group] * kLog2e : 0.f;
  Held<DP> q;
  q.load(qs + row_block * BLOCK);
  q.template wait<false>();
  const Score score(c);
  f32x16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) o[d] = zeros();
  // Of the lane's row: o is sum exp2(s) v times 2^offset, total sum exp2(s) times 2^(offset - 40).
  float offset = 1e9f, total = 0.f;
  const char *const from[2] = {ks, vs};
  const uint32_t to = lds_address(&lds[0][group][0]);
  if (begin + group < end) Blocks<DP, 2>(from, key_block + begin + group, to).all();
  int parity = 0;
#pragma unroll 1
  for (int pair = begin; pair < end; pair += 2, parity ^= 1) {
    const int step = pair + group, j0 = step * kKeys;
    arrived();
    if (step + 2 < end) Blocks<DP, 2>(from, key_block + step + 2, to + (uint32_t)((1 - parity) * 4 * BLOCK)).all();
    if (step >= end || !mine.meets(j0, j0 + kKeys)) continue;
    const int ek = scalar(ex.k + key_block + step), ev = scalar(ex.v + key_block + step);
    const char *const keys = lds[parity][group], *const values = keys + BLOCK;
    f32x16 s[1];
    products<DP, 1, AHEAD>(keys, {&q}, s, Nothing{});
    const float factor = unscaled(score.factor, eq, ek);
    const bool whole = mine.covers(j0, j0 + kKeys);
    float p[16], most = kNone;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      p[v] = s[0][v];
      if (!PLAIN) {
        p[v] *= factor;
        if (score.capped) p[v] = score.top * tanh_of(p[v]);
        p[v] -= slope * fabsf((float)(near - (j0 + key_of(v, half))));
      }
    }
    if (!whole)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int j = j0 + key_of(v, half);
        p[v] = j >= lo && j < hi ? p[v] : kNone;
      }
#pragma unroll
    for (int v = 0; v < 16; ++v) most = fmaxf(most, p[v]);
    most = fmaxf(most, other_half(most));
    if (PLAIN) most *= factor;
    // exp2(s + shift) is the other operand, to the scale of the block's values.  A row's offset follows the largest p v that it has, not what its
    // neighbours see or a large value of which it takes next to nothing: it is lowered where the operand would pass 2^15, to 2^9, so that most steps leave
    // the sums alone.
    float shift = offset - (float)ev;
    if (__any(most + shift > 15.f)) {
      const float lower = most + shift > 15.f ? 9.f - most + (float)ev : offset, fade = __builtin_amdgcn_exp2f(fmaxf(lower - offset, -200.f));
      total *= fade;
      multiply(o, fade);
      offset = lower;
      shift = offset - (float)ev;
    }
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      p[v] = __builtin_amdgcn_exp2f(PLAIN ? __builtin_fmaf(p[v], factor, shift) : p[v] + shift);
      sum += p[v];
    }
    total = __builtin_fmaf(sum, __builtin_ldexpf(1.f, ev - 40), total);
    // the second half's operands while the first half is multiplied
    Weights w;
    static_for<4>([&](auto n) { w.set<decltype(n)::value>(p[2 * decltype(n)::value], p[2 * decltype(n)::value + 1]); });
    add_product<DP, AHEAD>(o, values, w, [&](auto place) {
      spread<decltype(place)::value, 0, 3 * DP / 32 - 1, 4>([&](auto k) {
        constexpr int n = 4 + decltype(k)::value;
        w.set<n>(p[2 * n], p[2 * n + 1]);
      });
    });
  }
  total += other_half(total);
  // to a maximum with total in [1, 2), and o to the same
  const int above = (int)(bits_of(total) >> 23) - 127;
  const float top = total == 0.f ? kNone : (float)(40 + above) - offset;
  total = __builtin_ldexpf(total, -above);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = __builtin_ldexpf(o[d][v], -40 - above);
  // the second group's rows to the first
  __syncthreads();
  f32x4 *const room_o = reinterpret_cast<f32x4 *>(&lds[0][0][0]) + wave * (DP / 8 * 64);
  if (group == 1) {
    if (half == 0) {
      marks[0][wave * 32 + lane] = top;
      marks[1][wave * 32 + lane] = total;
    }
#pragma unroll
    for (int e = 0; e < DP / 8; ++e)
      room_o[e * 64 + lane] = f32x4{o[e / 4][e % 4 * 4], o[e / 4][e % 4 * 4 + 1], o[e / 4][e % 4 * 4 + 2], o[e / 4][e % 4 * 4 + 3]};
  }
  __syncthreads();
  if (group == 1 || !live) return;
  const float other_top = marks[0][wave * 32 + lane % 32], other_total = marks[1][wave * 32 + lane % 32];
  const float joined = fmaxf(top, other_top), base = joined == kNone ? 0.f : joined;
  const float mine_by = __builtin_amdgcn_exp2f(top - base), other_by = __builtin_amdgcn_exp2f(other_top - base);
  total = total * mine_by + other_total * other_by;
#pragma unroll
  for (int e = 0; e < DP / 8; ++e) {
    const f32x4 x = room_o[e * 64 + lane];
#pragma unroll
    for (int n = 0; n < 4; ++n) o[e / 4][e % 4 * 4 + n] = o[e / 4][e % 4 * 4 + n] * mine_by + x[n] * other_by;
  }
  float *row;
  const float by = row_end(c, pieces, out, stat, b, g, r, piece, joined, total, half == 0, row);
  if (row) store_sums(o, row, c.dim, by);
}

// ------------------------------------------------------------------------------ backward

// The unit of the sum of a lane's row or key, of gradients times what has exponent `other`: the step's largest gradient has to stay below 2^15 in it (the
// smallest ones lower, so that the factor is a number).  Where one has to be lowered it becomes less than 2^8, and so do those of more than 2^11, so that
// it seldom has to.  (A floor of 2^-32 of the largest.  To 2^6 the backward pass of 4 096 tokens of 16 heads of 128 takes 738 us, to 2^10 749, and so 741.)
__device__ __forceinline__ int gradient_unit(float most, int other, int unit, bool &lowers) {
  const int field = (int)(bits_of(fmaxf(most, other_half(most))) >> 23), limit = field == 0 || field == 255 ? INT32_MAX : 141 - max(field, 15) + other;
  lowers = __any(unit > limit);
  return lowers && unit > limit - 4 ? min(unit, limit - 7) : unit;
}
// The factor that brings such a gradient to it; a sum of nothing but zeros so far has none.
__device__ __forceinline__ float to_unit(int unit, int other) { return __builtin_ldexpf(1.f, unit == kNoUnit ? 0 : min(unit - other, 126)); }

// p times 2^x, for shift = x - the row's statistic, and the derivative of the cap, from a product.
template <bool PLAIN>
__device__ __forceinline__ float weight(const Score &score, float product, float factor, float bias, float shift, float &slope) {
  if (PLAIN) return __builtin_amdgcn_exp2f(__builtin_fmaf(product, factor, shift));
  float t = product * factor;
  slope = 1.f;
  if (score.capped) {
    t = tanh_of(t);
    slope = __builtin_fmaf(-t, t, 1.f);
    t *= score.top;
  }
  return __builtin_amdgcn_exp2f((t - bias) + shift);
}

// Whether two waves share a SIMD, in 256 registers each; longer heads have all 512, their sums and held operands among those that only matrix instructions work on.  With
// 96 columns two are faster where cap or bias are vector work to hide (2 x 1 777 tokens, documents, 6 heads on 3 of 72, the whole backward pass 145 us and 155), and slower
// without (4 096 tokens, 16 heads on 4 of 96, 626 and 611).
template <int DP, bool PLAIN>
constexpr bool kTwoWaves = DP <= 64 || (DP <= 96 && !PLAIN);

// 128 rows a workgroup, as forward_kernel; in LDS a step's keys, values and keys transposed.
template <int DP, bool PLAIN>
__global__ __launch_bounds__(kThreads, (kTwoWaves<DP, PLAIN>) ? 2 : 1) void dq_kernel(const Call c, const char *qs, const char *ds_, const char *ks, const char *vs, const char *kts,
                                                                        const Exponents ex, const Row *rows, float *dq, int64_t stride, int tiles, int pieces) {
  constexpr int BLOCK = (int)block_size(DP), AHEAD = DP > 64 && kTwoWaves<DP, PLAIN> ? 2 : 3;
  constexpr bool TWO = kTwoWaves<DP, PLAIN>;
  __shared__ __align__(16) char lds[2][3 * BLOCK];
  __shared__ int room[4][4];
  const int heads = c.batch * c.key_heads;
  const int bg = (int)blockIdx.x % heads, rest = (int)blockIdx.x / heads;
  const int b = bg / c.key_heads, g = bg % c.key_heads, tile = tiles - 1 - rest % tiles, piece = rest / tiles;
  const int lane = threadIdx.x % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int r = tile * kRows + wave * 32 + lane % 32;
  const bool live = r < c.rows;
  const Row row = rows[(int64_t)bg * c.rows + (live ? r : 0)];
  const int near = c.nearest(c.own(b, (live ? r : 0) / c.group), row.lo, row.hi);
  Hull mine;
  mine.of(row.lo, row.hi, live);
  const Hull all = mine.all(room);
  const int first = all.first(), steps = all.steps();
  if (__syncthreads_or(ex.bad_rows(bg, tile * (kRows / 32), first, steps))) return;
  const int begin = first + (int)((int64_t)steps * piece / pieces), end = first + (int)((int64_t)steps * (piece + 1) / pieces);
  const int block = min(tile * (kRows / 32) + wave, ex.row_blocks - 1);
  const int64_t row_block = (int64_t)bg * ex.row_blocks + block, key_block = (int64_t)bg * ex.key_blocks;
  const int eq = scalar(ex.q + row_block), ed = scalar(ex.d + row_block);
  const float slope = !PLAIN && c.slopes ? c.slopes[g * c.group + (live ? r : 0) % c.group] * kLog2e : 0.f;
  // a row that sees nothing has whatever statistic
  const bool some = live && row.lo < row.hi;
  const float stat = some ? row.stat : 0.f, delta = some ? row.delta : 0.f;
  Held<DP> q, d;
  q.load(qs + row_block * BLOCK);
  d.load(ds_ + row_block * BLOCK);
  d.alternate();
  const float sign = lane % 2 ? -1.f : 1.f;
  q.template wait<!TWO>();
  d.template wait<!TWO>();
  const Score score(c);
  f32x16 sum[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) sum[e] = zeros();
  int unit = kNoUnit;  // sum is times 2^unit, of the lane's row
  const char *const from[3] = {ks, vs, kts};
  const uint32_t to = lds_address(&lds[0][0]);
  if (begin < end) Blocks<DP, 3>(from, key_block + begin, to).all();
#pragma unroll 1
  for (int step = begin; step < end; ++step) {
    const int slot = (step - begin) & 1, j0 = step * kKeys;
    const int ek = scalar(ex.k + key_block + step), ev = scalar(ex.v + key_block + step);
    arrived();
    // the last step fetches itself again
    const Blocks<DP, 3> next(from, key_block + min(step + 1, end - 1), to + (uint32_t)((1 - slot) * 3 * BLOCK));
    if (TWO && !mine.meets(j0, j0 + kKeys)) {  // longer heads: the sums would move at every step for it
      next.all();
      continue;
    }
    keep<!TWO>(sum);
    const float factor = unscaled(score.factor, eq, ek), d_factor = __builtin_ldexpf(sign, -(ed + ev));
    float p[16], cap[16], ds[16];
    f32x16 s[2];
    auto tile = [&](auto whole_c) {
      constexpr bool WHOLE = decltype(whole_c)::value;
      products<DP, 2, AHEAD>(lds[slot], {&q, &d}, s, [&](auto place) {
        constexpr int FIRST = 3 * DP / 16;
        spread<decltype(place)::value, 0, FIRST, decltype(next)::kCount>([&](auto f) { next.template one<decltype(f)::value>(); });
        spread<decltype(place)::value, FIRST + 2, FIRST - 2, 16>([&](auto v_c) {
          constexpr int v = decltype(v_c)::value;
          const int j = j0 + key_of(v, half);
          p[v] = weight<PLAIN>(score, s[0][v], factor, PLAIN ? 0.f : slope * fabsf((float)(near - j)), -stat, cap[v]);
          if (!WHOLE) p[v] = ((j >= row.lo) & (j < row.hi)) ? p[v] : 0.f;
        });
      });
    };
    if (mine.covers(j0, j0 + kKeys)) tile(std::true_type{});
    else tile(std::false_type{});
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      ds[v] = p[v] * __builtin_fmaf(s[1][v], d_factor, -delta);
      if (!PLAIN) ds[v] *= cap[v];
    }
    float most = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) most = fmaxf(most, fabsf(ds[v]));
    bool lowers;
    const int new_unit = gradient_unit(most, ek, unit, lowers);
    if (lowers) {
      multiply(sum, __builtin_ldexpf(1.f, max(new_unit - unit, -200)));
      keep<!TWO>(sum);
      unit = new_unit;
    }
    const float scale = to_unit(unit, ek);
    Weights w;
    auto set = [&](auto n_c) {
      constexpr int n = decltype(n_c)::value;
      w.set<n>(ds[2 * n] * scale, ds[2 * n + 1] * scale);
    };
    static_for<4>(set);
    add_product<DP, AHEAD>(sum, lds[slot] + 2 * BLOCK, w,
                           [&](auto place) { spread<decltype(place)::value, 0, 3 * DP / 32 - 1, 4>([&](auto k) { set(IC<4 + decltype(k)::value>{}); }); });
  }
  arrived();  // what the last step has fetched
  if (!live) return;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
#pragma unroll
    for (int v = 0; v < 16; ++v) sum[e][v] = __builtin_ldexpf(sum[e][v], unit == kNoUnit ? 0 : -unit);
  store_sums(sum, dq + piece * stride + c.query_at(b, g, r), c.dim, c.scale);
}

// 128 keys a workgroup, 32 a wave; steps of 32 rows: in LDS queries, gradients, both transposed, and what Info says of the rows.
template <int DP, bool PLAIN>
__global__ __launch_bounds__(kThreads, DP <= 64 ? 2 : 1) void dkv_kernel(const Call c, const char *qs, const char *ds_, const char *qts, const char *dts, const char *ks,
                                                                         const char *vs, const Exponents ex, const char *info,
                                                                         float *dk, float *dv, float *parts, int tiles, int pieces) {
  constexpr int BLOCK = (int)block_size(DP), SLOT = 4 * BLOCK + kInfoBytes, AHEAD = DP <= 64 ? 1 : 3;
  __shared__ __align__(16) char lds[2][SLOT];
  __shared__ int range[2];
  // Earlier keys, which more rows see in a causal pass, first.
  const int heads = c.batch * c.key_heads, bg = (int)blockIdx.x % heads, piece = (int)blockIdx.x / heads % pieces, tile = (int)blockIdx.x / heads / pieces;
  const int b = bg / c.key_heads, g = bg % c.key_heads;
  const int lane = threadIdx.x % 64, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int tile_lo = tile * kRows, tile_hi = min(c.tk, tile_lo + kRows);
  if (__syncthreads_or(ex.bad_keys(bg, tile_lo / 32, tile_lo, tile_hi))) return;
  const int64_t row_block = (int64_t)bg * ex.row_blocks;
  // The blocks of rows that see one of the keys; a piece has every pieces-th of them, from the last on, which in a causal pass all tiles see: a piece's tiles
  // of one head, on one XCD where heads times pieces are a multiple of 8, go through the same blocks together and find them in its L2.  (4 096 x 16
  // heads of 128 on 4, causal: 443 MiB from memory and 408 us; pieces one behind the other, of each tile's rows, 1 985 MiB and 426, the whole backward pass 789 us and 747;
  // pieces one behind the other, of all rows, leave a third of the CUs without work: 685, or 475 with tiles from both ends in one workgroup.)
  if (threadIdx.x == 0) range[0] = ex.row_blocks, range[1] = 0;
  __syncthreads();
  {
    int lo = ex.row_blocks, hi = 0;
    for (int e = threadIdx.x; e < ex.row_blocks; e += kThreads)
      if (ex.hulls[row_block + e].meets(tile_lo, tile_hi)) lo = min(lo, e), hi = max(hi, e + 1);
    atomicMin(&range[0], lo);
    atomicMax(&range[1], hi);
  }
  __syncthreads();
  const int first = __builtin_amdgcn_readfirstlane(range[0]), steps = max(0, __builtin_amdgcn_readfirstlane(range[1]) - first);
  const int j0 = tile_lo + wave * 32, j = j0 + lane % 32;
  const bool live = j < c.tk;
  const int64_t key_block = (int64_t)bg * ex.key_blocks + min(tile * (kRows / 32) + wave, ex.key_blocks - 1);
  const int ek = scalar(ex.k + key_block), ev = scalar(ex.v + key_block);
  Held<DP> k, v;
  k.load(ks + key_block * BLOCK);
  v.load(vs + key_block * BLOCK);
  v.alternate();
  const float sign = lane % 2 ? -1.f : 1.f;
  k.template wait<(DP > 64)>();
  v.template wait<(DP > 64)>();
  const Score score(c);
  f32x16 dks[DP / 32], dvs[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) dks[e] = dvs[e] = zeros();
  int unit = kNoUnit, unit_v = kNoUnit;  // dks are times 2^unit, dvs times 2^unit_v, of the lane's key
  const char *const from[4] = {qs, ds_, qts, dts};
  const uint32_t to = lds_address(&lds[0][0]);
  auto fetch_info = [&](int step, int slot) {
    if (wave == 0) fetch<0, false>(__builtin_amdgcn_readfirstlane(to + (uint32_t)(slot * SLOT + 4 * BLOCK)), uniform(info + (row_block + step) * kInfoBytes));
  };
  auto hull_of = [&](int step, Hull &seen) {
    seen.lo = scalar(&ex.hulls[row_block + step].lo);
    seen.hi = scalar(&ex.hulls[row_block + step].hi);
    seen.inner_lo = scalar(&ex.hulls[row_block + step].inner_lo);
    seen.inner_hi = scalar(&ex.hulls[row_block + step].inner_hi);
  };
  // the first block from `step` on that sees one of the workgroup's keys; others may be some that cannot be split, of which nothing is stored
  auto next_of = [&](int step) {
    Hull seen;
    for (; step >= first; step -= pieces) {
      hull_of(step, seen);
      if (seen.meets(tile_lo, tile_hi)) break;
    }
    return step;
  };
  const int last = first + steps - 1;
  int step = next_of(last - (last + pieces - piece) % pieces), slot = 0;
  if (step >= first) {
    Blocks<DP, 4>(from, row_block + step, to).all();
    fetch_info(step, 0);
  }
#pragma unroll 1
  for (int next; step >= first; step = next, slot ^= 1) {
    const int eq = scalar(ex.q + row_block + step), ed = scalar(ex.d + row_block + step);
    Hull seen;
    hull_of(step, seen);
    next = next_of(step - pieces);
    arrived();
    // the last step fetches itself again
    const Blocks<DP, 4> coming(from, row_block + (next >= first ? next : step), to + (uint32_t)((1 - slot) * SLOT));
    fetch_info(next >= first ? next : step, 1 - slot);
    keep<(DP > 64)>(dks);
    keep<(DP > 64)>(dvs);
    if (DP <= 64 && !seen.meets(j0, j0 + 32)) {  // longer heads: the sums would move at every step for it
      coming.all();
      continue;
    }
    const char *const at = lds[slot];
    const float factor = unscaled(score.factor, eq, ek), d_factor = __builtin_ldexpf(sign, -(ed + ev));
    // p enters the sum of dv times this, 2^60 until the key's first share says what it is to be.  (As part of its exponent it would cost nothing, but
    // the exponents of the shares that count would be rounded at its size: dk and dv of documents with distances 7.7e-7 off, and so 2.9e-7 to 3.7e-7.)
    auto held_by = [&](int u) { return u == kNoUnit ? kFirstHeld : min(max(u - ed, -126), 126); };
    const float scale = __builtin_ldexpf(1.f, held_by(unit_v));
    const float *const of = reinterpret_cast<const float *>(at + 4 * BLOCK) + 4 * half;
    auto four = [&](int array, int q) { return *reinterpret_cast<const f32x4 *>(of + 32 * array + 8 * q); };
    float p[16], cap[16], ds[16], most = 0.f;
    f32x16 s[2];
    Weights w;
    auto tile = [&](auto whole_c) {
      constexpr bool WHOLE = decltype(whole_c)::value;
      // all at once, or, where the registers are full, as they are needed
      constexpr bool LATE = !PLAIN && DP == 64;
      f32x4 shift[LATE ? 1 : 4];
      if constexpr (!LATE) static_for<4>([&](auto q) { shift[decltype(q)::value] = -four(kStat, decltype(q)::value); });
      products<DP, 2, AHEAD>(at, {&k, &v}, s, [&](auto place) {
        constexpr int FIRST = 3 * DP / 16;
        spread<decltype(place)::value, 0, FIRST, decltype(coming)::kCount>([&](auto f) { coming.template one<decltype(f)::value>(); });
        spread<decltype(place)::value, FIRST + 2, FIRST - 4, 16>([&](auto x_c) {
          constexpr int x = decltype(x_c)::value, q = x / 4, e = x % 4;
          if constexpr (LATE && e == 0) shift[0] = -four(kStat, q);
          float bias = 0.f;
          if (!PLAIN && c.slopes) bias = of[32 * kSlope + 8 * q + e] * fabsf(of[32 * kNear + 8 * q + e] - (float)j);
          p[x] = weight<PLAIN>(score, s[0][x], factor, bias, shift[LATE ? 0 : q][e], cap[x]);
          if (!WHOLE) {
            const int lo = (int)bits_of(of[32 * kLo + 8 * q + e]), hi = (int)bits_of(of[32 * kHi + 8 * q + e]);
            p[x] = ((j >= lo) & (j < hi)) ? p[x] : 0.f;
          }
          if constexpr (x % 2) most = fmaxf(fmaxf(most, p[x - 1]), p[x]);
        });
        // two values behind
        spread<decltype(place)::value, FIRST + 4, FIRST - 4, 8>([&](auto n_c) {
          constexpr int n = decltype(n_c)::value;
          w.set<n>(p[2 * n] * scale, p[2 * n + 1] * scale);
        });
      });
    };
    if (seen.covers(j0, j0 + 32)) tile(std::true_type{});
    else tile(std::false_type{});
    // A key's first share sets its unit.  Shares that pass what fp16 holds, or that are not held as the sum needs them, lower it so that they become less than 2^8, and
    // of the wave's other keys that of those of more than 2^11, so that this is seldom; a first share too small for its digits raises it as far.  A unit follows the largest
    // p do that its key has had, whatever the rows give to others.
    most = fmaxf(most, other_half(most));
    asm("" : "+v"(unit_v));  // what follows from it is computed again, not kept all along
    const int held = held_by(unit_v);
    const float passes = unit_v - ed > 126 && unit_v != kNoUnit ? 0.f : __builtin_ldexpf(65000.f, -held);
    const bool first = unit_v == kNoUnit && most > 0.f, small = first && most < __builtin_ldexpf(0.25f, -kFirstHeld);
    int next_unit = first ? held + ed : unit_v;
    if (__any(most > passes || small)) {
      const bool moves = most > passes * 0x1p-5f || small;
      const int to = moves ? min(min(unit_v - ed, 126), 134 - (int)(bits_of(most) >> 23)) : held;
      static_for<8>([&](auto n_c) {
        constexpr int n = decltype(n_c)::value;
        w.set<n>(__builtin_ldexpf(p[2 * n], to), __builtin_ldexpf(p[2 * n + 1], to));
      });
      if (moves) next_unit = to + ed;
      multiply(dvs, __builtin_ldexpf(1.f, max(next_unit - unit_v, -200)));
      keep<(DP > 64)>(dvs);
    }
    unit_v = next_unit;
    // While dv is summed: ds, the unit that dk's sum takes for it, and ds as that product's operand.
    f32x4 delta[4];
    static_for<4>([&](auto q) { delta[decltype(q)::value] = four(kDelta, decltype(q)::value); });
    constexpr int PLACES = 3 * DP / 16, HALF = PLACES / 2;
    int new_unit = unit;
    float to_sum = 1.f;
    float largest = 0.f;
    bool lowers = false;
    Weights wd;
    add_product<DP, AHEAD>(dvs, at + 3 * BLOCK, w, [&](auto place) {
      constexpr int at_place = decltype(place)::value;
      spread<at_place, 0, HALF - 1, 16>([&](auto x_c) {
        constexpr int x = decltype(x_c)::value;
        ds[x] = p[x] * __builtin_fmaf(s[1][x], d_factor, -delta[x / 4][x % 4]);
        if (!PLAIN) ds[x] *= cap[x];
        if constexpr (x % 2) largest = fmaxf(fmaxf(largest, fabsf(ds[x - 1])), fabsf(ds[x]));
      });
      if constexpr (at_place == HALF - 1) {
        new_unit = gradient_unit(largest, eq, unit, lowers);
        to_sum = to_unit(new_unit, eq);
      }
      spread<at_place, HALF, PLACES - HALF, 8>([&](auto n_c) {
        constexpr int n = decltype(n_c)::value;
        wd.set<n>(ds[2 * n] * to_sum, ds[2 * n + 1] * to_sum);
      });
    });
    if (lowers) {
      multiply(dks, __builtin_ldexpf(1.f, max(new_unit - unit, -200)));
      keep<(DP > 64)>(dks);
      unit = new_unit;
    }
    add_product<DP, AHEAD>(dks, at + 2 * BLOCK, wd, Nothing{});
  }
  arrived();  // what the last step has fetched
  if (!live) return;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      dks[e][x] = __builtin_ldexpf(dks[e][x], unit == kNoUnit ? 0 : -unit);
      dvs[e][x] = __builtin_ldexpf(dvs[e][x], -unit_v);
    }
  const int64_t all = (int64_t)c.batch * c.tk * c.key_heads * c.dim, key = c.key_at(b, g, j);
  float *const to_k = pieces > 1 ? parts + (int64_t)piece * 2 * all : dk, *const to_v = pieces > 1 ? parts + ((int64_t)piece * 2 + 1) * all : dv;
  if (to_k) store_sums(dks, to_k + key, c.dim, c.scale);
  if (to_v) store_sums(dvs, to_v + key, c.dim, 1.f);
}

// ------------------------------------------------------------------------------ host

int columns_of(int dim) { return (dim + 31) / 32 * 32; }

template <class F>
void with_columns(int dim, const F &f) {
  if (dim <= 32) f(IC<32>{});
  else if (dim <= 64) f(IC<64>{});
  else if (dim <= 96) f(IC<96>{});
  else f(IC<128>{});
}
int blocks_of(int64_t rows) { return (int)((rows + 31) / 32); }

// Scratch, handed out piece by piece on 256-byte bounds.
struct Scratch {
  char *at;
  size_t used;
  char *take(size_t bytes) {
    char *p = at + used;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};

struct Layout {
  char *q, *d, *k, *v, *qt, *dt, *kt, *vt, *info;
  int *eq, *ed, *ek, *ev;
  Hull *hulls;
  int2 *seen;
  Layout(const Call &c, bool backward, Scratch &s) {
    const int64_t heads = (int64_t)c.batch * c.key_heads, rows = heads * blocks_of(c.rows), keys = heads * blocks_of(c.tk);
    const size_t row_bytes = (size_t)rows * block_size(columns_of(c.dim)), key_bytes = (size_t)keys * block_size(columns_of(c.dim));
    q = s.take(row_bytes);
    k = s.take(key_bytes);
    d = backward ? s.take(row_bytes) : nullptr;
    v = backward ? s.take(key_bytes) : nullptr;
    qt = backward ? s.take(row_bytes) : nullptr;
    dt = backward ? s.take(row_bytes) : nullptr;
    kt = backward ? s.take(key_bytes) : nullptr;
    vt = backward ? nullptr : s.take(key_bytes);
    info = backward ? s.take((size_t)rows * kInfoBytes) : nullptr;
    eq = (int *)s.take(rows * 4);
    ek = (int *)s.take(keys * 4);
    ev = (int *)s.take(keys * 4);
    ed = backward ? (int *)s.take(rows * 4) : nullptr;
    hulls = backward ? (Hull *)s.take(rows * sizeof(Hull)) : nullptr;
    // All spans in every workgroup of keys are quadratic: forward, documents of 1 024, 131 072 tokens of 4 heads of 64 3 134 us and here 570; of 512, 4 096 tokens
    // 59.9 and 57.7, 2 048 tokens 63.8 and with the launch 65.9.
    seen = c.spans && c.tq > kSpansReadByAll ? (int2 *)s.take(c.batch * sizeof(int2)) : nullptr;
  }
};

void pack(const Call &c, Pack &p, int2 *seen, hipStream_t s) {
  p.seen = seen;
  if (seen) hipLaunchKernelGGL(seen_kernel, dim3((unsigned)c.batch), dim3(1024), 0, s, c, seen);
  const int heads = c.batch * c.key_heads;
  int groups = 0;
  p.row_blocks = blocks_of(c.rows);
  p.key_blocks = blocks_of(c.tk);
  for (int i = 0; i < p.n_jobs; ++i) {
    p.jobs[i].first = groups;
    groups += heads * (p.jobs[i].of_rows ? p.row_blocks : p.key_blocks);
  }
  with_columns(c.dim, [&](auto dp) { hipLaunchKernelGGL((pack_kernel<decltype(dp)::value>), dim3((unsigned)groups), dim3(kThreads), 0, s, c, p); });
}

// Exponents::least_sum: elements of a block are less than 2^15 times 2^-exponent
int least_sum(const Call &c) {
  int exponent;
  (void)frexp((double)c.scale * c.dim, &exponent);   // 2^exponent is more
  return exponent + 30 - 18;
}

}  // namespace

bool pair_suits(const Call &c, bool backward) {
  const char *e = getenv("TINYFLOW_SPLIT");
  if (e && e[0] == '0') return false;
  const float factor = c.cap > 0.f ? c.scale / c.cap : c.scale;
  if (c.dim > 128 || !(factor > 0x1p-40f && factor < 0x1p40f)) return false;
  // Below these splitting costs more than it saves.  Microseconds of a call, fp32 kernels / these, one head: forward, 33 x 33 of 64 12 / 16, 128 x 128 of 32
  // 13 / 15, 33 x 257 of 32 24 / 18, 128 x 128 of 64 21 / 17, 64 x 64 of 128 20 / 18; backward, 64 x 64 of 32 25 / 30, 33 x 33 of 64 36 / 32, 33 x 257 of 32
  // 36 / 34, 8 x 1024 of 32 30 / 35 and of 64 43 / 37.
  if (!backward && (int64_t)c.tk * c.dim < 8192) return false;
  if (backward && ((int64_t)std::max(c.rows, c.tk) * c.dim <= 2048 || (c.dim <= 32 && std::min(c.rows, c.tk) < 32))) return false;
  // the planes are written by one launch, a block a workgroup
  if ((int64_t)c.batch * c.key_heads * (blocks_of(c.rows) + (int64_t)blocks_of(c.tk)) * 2 >= 1 << 24) return false;
  return true;
}

size_t pair_bytes(const Call &c, bool backward) {
  Scratch s = {nullptr, 0};
  Layout l(c, backward, s);
  return s.used;
}

Exponents pair_forward(const Call &c, float *out, float *stat, const Pieces &pieces, int tiles, char *scratch, hipStream_t s) {
  Scratch of = {scratch, 0};
  const Layout l(c, false, of);
  Pack p = {};
  p.n_jobs = 3;
  p.jobs[0] = Job{c.q, true, false, l.q, nullptr, l.eq, 0};
  p.jobs[1] = Job{c.k, false, false, l.k, nullptr, l.ek, 0};
  p.jobs[2] = Job{c.v, false, true, nullptr, l.vt, l.ev, 0};
  pack(c, p, l.seen, s);
  const Exponents ex = {l.eq, nullptr, l.ek, l.ev, nullptr, p.row_blocks, p.key_blocks, least_sum(c)};
  const unsigned groups = (unsigned)((int64_t)c.batch * c.key_heads * tiles * pieces.count);
  const bool plain = !c.slopes && c.cap == 0.f;
  with_columns(c.dim, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    hipLaunchKernelGGL((plain ? forward_kernel<DP, true> : forward_kernel<DP, false>), dim3(groups), dim3(2 * kThreads), 0, s, c, l.q, l.k, l.vt, ex, out, stat, pieces, tiles);
  });
  return ex;
}

Exponents pair_backward(const Call &c, const float *out, const float *stat, const float *dout, Row *rows, const Gradients &to, int row_tiles, int key_tiles,
                        char *scratch, hipStream_t s) {
  Scratch of = {scratch, 0};
  const Layout l(c, true, of);
  Pack p = {};
  p.n_jobs = 4;
  const bool keys = to.dk || to.dv;
  p.jobs[0] = Job{c.q, true, true, l.q, keys ? l.qt : nullptr, l.eq, 0};
  p.jobs[1] = Job{dout, true, true, l.d, keys ? l.dt : nullptr, l.ed, 0};
  p.jobs[2] = Job{c.k, false, true, l.k, to.dq ? l.kt : nullptr, l.ek, 0};
  p.jobs[3] = Job{c.v, false, true, l.v, nullptr, l.ev, 0};
  p.out = out;
  p.stat = stat;
  p.rows = rows;
  p.info = (float *)l.info;
  p.hulls = l.hulls;
  pack(c, p, l.seen, s);
  const Exponents ex = {l.eq, l.ed, l.ek, l.ev, l.hulls, p.row_blocks, p.key_blocks, least_sum(c)};
  const bool plain = !c.slopes && c.cap == 0.f;
  const int heads = c.batch * c.key_heads;
  with_columns(c.dim, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if (to.dq)
      hipLaunchKernelGGL((plain ? dq_kernel<DP, true> : dq_kernel<DP, false>), dim3((unsigned)(heads * row_tiles * to.row_pieces)), dim3(kThreads), 0, s, c, l.q, l.d, l.k,
                         l.v, l.kt, ex, rows, to.dq, to.row_stride, row_tiles, to.row_pieces);
    if (keys)
      hipLaunchKernelGGL((plain ? dkv_kernel<DP, true> : dkv_kernel<DP, false>), dim3((unsigned)(heads * to.pieces * key_tiles)), dim3(kThreads), 0, s, c, l.q, l.d, l.qt,
                         l.dt, l.k, l.v, ex, l.info, to.dk, to.dv, to.parts, key_tiles, to.pieces);
  });
  return ex;
}

}  // namespace attention
}  // namespace tf
