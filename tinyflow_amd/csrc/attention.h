// What the attention kernels share: the view of a call's arrays, which keys a query sees, and how a score comes out of a product.
//
//   s_ij = cap tanh(scale q_i k_j / cap) - slope |a_i - j|, seen keys only, a_i = i + Tk - Tq or as given;   without a cap s = scale q k
//   o_i = sum_j p_ij v_j, p_ij = exp(s_ij - stat_i), stat_i = log sum_j exp(s_ij);    nothing seen: o = 0, stat = -inf
//   backward: ds_ij = p_ij (do_i v_j - delta_i) cap'_ij scale, delta_i = do_i o_i
//             dq_i = sum_j ds_ij k_j, dk_j = sum_i ds_ij q_i, dv_j = sum_i p_ij do_i
//
// Scores are kept times log2 e: p is then one exp2 of a difference.  Every mask is an interval of keys for each query, [first, last): a document's, a
// prefix's, a window's, the used part of a cache, and the keys up to the query's own with `causal`.
//
// The query heads that share a key head are rows of one matrix: row r of key head g is query r / group, head g * group + r % group.  A
// tile of rows then reads a key once for all of them.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace tf {
namespace attention {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));  // rows of any length start anywhere: 16-byte accesses on 4-byte alignment
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct Call {
  const float *q, *k, *v;
  const float *spans;      // [queries, span_width], of each batch entry where span_stride is not 0
  const float *slopes;     // of each query head
  int64_t span_stride;
  int span_width;          // 3: with the key that a query stands at
  int batch, tq, tk, heads, key_heads, group, dim;
  int rows;                // tq * group: of a key head
  float scale, cap;        // cap 0: none
  bool causal;

  __device__ inline int64_t query_at(int b, int g, int r) const {  // of row r of key head g; also of o, do, dq
    return (((int64_t)b * tq + r / group) * heads + g * group + r % group) * dim;
  }
  __device__ inline int64_t key_at(int b, int g, int j) const { return (((int64_t)b * tk + j) * key_heads + g) * dim; }
  __device__ inline int64_t stat_at(int b, int g, int r) const { return ((int64_t)b * heads + g * group + r % group) * tq + r / group; }
  // The key that query i stands at: the keys' last ones are the queries' own, or what its span says.  (A NaN counts as far in front.)
  __device__ inline int own(int i, const float *span) const {
    const float given = span[span_width - 1];  // read in any case: behind a branch it would wait for all other loads
    return span_width < 3 ? i + tk - tq : (int)fminf(fmaxf(given, -0x1p24f), 0x1p24f);
  }
  __device__ inline const float *span_of(int b, int i) const { return spans + b * span_stride + span_width * (int64_t)i; }
  __device__ inline int own(int b, int i) const { return spans ? own(i, span_of(b, i)) : i + tk - tq; }
  // The keys that query i sees: [lo, hi), lo >= hi for none; and where it stands.
  __device__ inline void seen(int b, int i, int &lo, int &hi, int &at) const {
    lo = 0;
    hi = tk;
    at = i + tk - tq;
    if (spans) {
      const float *span = span_of(b, i);
      const float first = span[0], last = span[1];
      at = own(i, span);
      // key j is seen where first <= j < last; a NaN sees none
      if (!(first < last)) hi = 0;
      else {
        if (first > 0.f) lo = first < (float)tk ? (int)ceilf(first) : tk;
        if (last < (float)tk) hi = last > 0.f ? (int)ceilf(last) : 0;
      }
    }
    if (causal) hi = min(hi, at + 1);
  }
  __device__ inline void seen(int b, int i, int &lo, int &hi) const {
    int at;
    seen(b, i, lo, hi, at);
  }
  // Distances are counted from the nearest key that a query sees, so that they are as small as what they tell apart: the kernels' s lacks slope times the distance
  // of that key, from which all others are farther by as much.  It comes back with the statistic.  (With the distances themselves shares had the rounding of
  // the farthest: 1e-3 over 131 072 keys of which 1 000 are used.)
  __device__ static inline int nearest(int at, int lo, int hi) { return lo < hi ? min(max(at, lo), hi - 1) : at; }
  // log2 of a row's sum to its statistic, and back to what the backward kernels take from a score
  __device__ inline float statistic(int b, int g, int r, float log2_sum) const {
    const float x = log2_sum * kLn2;
    if (!slopes) return x;
    int lo, hi, at;
    seen(b, r / group, lo, hi, at);
    return fmaf(-slopes[g * group + r % group], (float)abs(at - nearest(at, lo, hi)), x);
  }
  __device__ inline float taken(int b, int g, int r, int lo, int hi, float statistic) const {
    if (!slopes) return statistic * kLog2e;
    const int at = own(b, r / group), away = abs(at - nearest(at, lo, hi));
    return (float)(((double)statistic + (double)slopes[g * group + r % group] * (double)away) * 1.4426950408889634);
  }
};

// tanh to a few steps of its own last place: near 0 the series, whose next term is 4e-3 x^12 of it, elsewhere from exp2, where 1 - e does
// not cancel.
__device__ inline float tanh_of(float x) {
  const float a = fabsf(x), e = __builtin_amdgcn_exp2f(-2.f * kLog2e * a), far = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
  const float y = x * x;
  float near = fmaf(y, -0.00886323552990219656f, 0.0218694885361552028f);
  near = fmaf(y, near, -0.0539682539682539683f);
  near = fmaf(y, near, 0.133333333333333333f);
  near = fmaf(y, near, -0.333333333333333333f);
  near = fmaf(y * a, near, a);
  return copysignf(a < 0.34f ? near : far, x);
}

// From a product to a score times log2 e, and back to the derivative of the cap.
struct Score {
  float factor;   // scale log2 e, or scale / cap
  float top;      // cap log2 e
  bool capped;
  __device__ inline explicit Score(const Call &c)
      : factor(c.cap > 0.f ? c.scale / c.cap : c.scale * kLog2e), top(c.cap * kLog2e), capped(c.cap > 0.f) {}
  __device__ inline float operator()(float product) const { return capped ? top * tanh_of(product * factor) : product * factor; }
};

// Finite or not, whatever the compiler assumes of comparisons.
__host__ __device__ inline bool finite(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) != 0x7f800000u; }

__device__ inline f32x4 load4(const float *p, int count) {
  if (count >= 4) return *reinterpret_cast<const f32x4u *>(p);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (count > 0) v[0] = p[0];
  if (count > 1) v[1] = p[1];
  if (count > 2) v[2] = p[2];
  return v;
}
__device__ inline void store4(float *p, int count, f32x4 v) {
  if (count >= 4) *reinterpret_cast<f32x4u *>(p) = v;
  else {
    if (count > 0) p[0] = v[0];
    if (count > 1) p[1] = v[1];
    if (count > 2) p[2] = v[2];
  }
}

// ------------------------------------------------------------------------------ what a wave and a workgroup see

constexpr int kThreads = 256, kRows = 128, kKeys = 32;  // of a workgroup; rows in the forward pass, keys in dkv; steps of the other axis
constexpr float kNone = -__builtin_inff();

__device__ inline float other_half(float v) {  // lane ^ 32
  const uint32_t bits = __builtin_bit_cast(uint32_t, v);
  const auto halves = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
  return __builtin_bit_cast(float, threadIdx.x % 64 < 32 ? halves[1] : halves[0]);
}

// Row of a 32 x 32 tile that a lane's v-th of 16 values stands for (the layout of the matrix instructions' sums), half = lane / 32.
constexpr int key_of(int v, int half) { return 8 * (v / 4) + 4 * half + v % 4; }

// The least and the greatest of what a wave's 32 columns, or a workgroup's 128, see, empty ones aside; inner: what all of them see.
struct Hull {
  int lo, hi, inner_lo, inner_hi;
  __device__ inline void of(int lo_, int hi_, bool live) {
    const bool some = live && lo_ < hi_;
    lo = some ? lo_ : INT32_MAX;
    hi = some ? hi_ : 0;
    inner_lo = some ? lo_ : INT32_MAX;
    inner_hi = some ? hi_ : 0;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) {
      lo = min(lo, __shfl_xor(lo, step));
      hi = max(hi, __shfl_xor(hi, step));
      inner_lo = max(inner_lo, __shfl_xor(inner_lo, step));
      inner_hi = min(inner_hi, __shfl_xor(inner_hi, step));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    inner_lo = __builtin_amdgcn_readfirstlane(inner_lo);
    inner_hi = __builtin_amdgcn_readfirstlane(inner_hi);
  }
  // over a workgroup's waves, through `room`
  template <int WAVES>
  __device__ inline Hull all(int (&room)[WAVES][4]) const {
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) room[wave][0] = lo, room[wave][1] = hi, room[wave][2] = inner_lo, room[wave][3] = inner_hi;
    __syncthreads();
    Hull h = *this;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      h.lo = min(h.lo, room[w][0]);
      h.hi = max(h.hi, room[w][1]);
      h.inner_lo = max(h.inner_lo, room[w][2]);
      h.inner_hi = min(h.inner_hi, room[w][3]);
    }
    h.lo = __builtin_amdgcn_readfirstlane(h.lo);
    h.hi = __builtin_amdgcn_readfirstlane(h.hi);
    return h;
  }
  __device__ inline bool meets(int from, int to) const { return lo < to && hi > from; }
  __device__ inline bool covers(int from, int to) const { return inner_lo <= from && inner_hi >= to; }
  // the steps of kKeys keys that it meets: [first, first + steps)
  __device__ inline int first() const { return lo < hi ? lo / kKeys : 0; }
  __device__ inline int steps() const { return lo < hi ? (hi + kKeys - 1) / kKeys - first() : 0; }
};

// Pieces of rows: [piece][row of all][dim] unnormalised sums and [piece][row of all] (maximum, sum); a row of all is (b, key head, row).
struct Pieces {
  float *sums;
  float2 *marks;
  int count;
  int64_t rows;  // of all
};

// Where a row's result or its piece is written, and what it is to be multiplied by.
__device__ inline float row_end(const Call &c, const Pieces &to, float *out, float *stat, int b, int g, int r, int piece, float top, float total,
                                bool writes_mark, float *&row) {
  if (to.count > 1) {
    const int64_t at = piece * to.rows + ((int64_t)b * c.key_heads + g) * c.rows + r;
    if (writes_mark) to.marks[at] = make_float2(top, total);
    row = to.sums + at * c.dim;
    return 1.f;
  }
  if (stat && writes_mark) stat[c.stat_at(b, g, r)] = total == 0.f ? kNone : c.statistic(b, g, r, top + __builtin_amdgcn_logf(total));
  row = out ? out + c.query_at(b, g, r) : nullptr;
  return total == 0.f ? 0.f : 1.f / total;
}

// What the backward kernels read of a row: its statistic in their terms (Call::taken), delta, and the keys that it sees.
struct Row {
  float stat, delta;
  int lo, hi;
};

// p and ds / scale from the products of queries and keys, and of gradients and values.
__device__ inline void gradient(const Score &score, float product, float dp, float bias, float stat, float delta, bool seen, float &p, float &ds) {
  float t = product * score.factor, slope = 1.f;
  if (score.capped) {
    t = tanh_of(t);
    slope = 1.f - t * t;
    t *= score.top;
  }
  p = seen ? __builtin_amdgcn_exp2f(t - bias - stat) : 0.f;
  ds = seen ? p * (dp - delta) * slope : 0.f;
}

// The sums of a tile's columns, `blocks` of 32: column 32 d + key_of(v, half) of the lane's row, times `by`.
template <int BLOCKS>
__device__ inline void store_sums(const f32x16 (&v)[BLOCKS], float *row, int dim, float by) {
  const int half = threadIdx.x % 64 / 32;
#pragma unroll
  for (int d = 0; d < BLOCKS; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 32 * d + 8 * q + 4 * half;
      if (c < dim) store4(row + c, dim - c, f32x4{v[d][4 * q] * by, v[d][4 * q + 1] * by, v[d][4 * q + 2] * by, v[d][4 * q + 3] * by});
    }
}

// ------------------------------------------------------------------------------ operands split into pairs (attention_pair.hip)

constexpr int kBad = INT32_MIN / 4;  // exponent of a block that cannot be split

// Of blocks of 32 rows, [b, key head][block]: exponents of queries, their gradients, keys and values, and what the block's rows see.  What a call does
// not have is null.
struct Exponents {
  const int *q, *d, *k, *v;
  const Hull *hulls;
  int row_blocks, key_blocks;

  // An element is off by up to 2^-39 of its block's largest value, which moves a score by up to 2^-39 of scale times the columns times the largest of both
  // blocks: what two exponents must add up to for a bound of 2^18 on that product, so 2^-21 on the error.  Queries and keys of a few units pass it by
  // 2^8 with 128 columns.
  int least_sum;

  // Whether what a (b, key head) has in the blocks of a tile cannot be computed on pairs, in the lanes that find out: the tile's four blocks of rows from
  // `first` on and the blocks of keys that they see.
  __device__ inline bool bad_rows(int64_t head, int first, int first_key, int n_keys) const {
    bool found = false;
    int least = INT32_MAX / 2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t at = head * row_blocks + min(first + e, row_blocks - 1);
      least = min(least, q[at]);
      if (d) found |= n_keys > 0 && d[at] == kBad;
    }
    for (int e = threadIdx.x; e < n_keys; e += blockDim.x) {
      const int64_t at = head * key_blocks + first_key + e;
      found |= first_key + e < key_blocks && (least + k[at] < least_sum || v[at] == kBad);
    }
    return found;
  }
  // A tile's four blocks of keys from `first` on, the keys [from, to), and the blocks of rows that see one of them.
  __device__ inline bool bad_keys(int64_t head, int first, int from, int to) const {
    bool bad_value = false, found = false;
    int least = INT32_MAX / 2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t at = head * key_blocks + min(first + e, key_blocks - 1);
      least = min(least, k[at]);
      bad_value |= v[at] == kBad;
    }
    for (int e = threadIdx.x; e < row_blocks; e += blockDim.x) {
      const int64_t at = head * row_blocks + e;
      found |= (least + q[at] < least_sum || d[at] == kBad || bad_value) && hulls[at].meets(from, to);
    }
    return found;
  }
  // Whether any tile of a (b, key head) may be such: either a query's or a key's exponent is below its share of the sum.  The fp32 kernels ask this first: of a head
  // without one they only see its exponents (dq of 4 096 x 16 heads of 128 5.3 us, 7.9 without).
  __device__ inline bool bad_head(int64_t head) const {
    const int share = least_sum >> 1;
    bool found = false;
    for (int e = threadIdx.x; e < row_blocks; e += blockDim.x) found |= q[head * row_blocks + e] < share || (d && d[head * row_blocks + e] == kBad);
    for (int e = threadIdx.x; e < key_blocks; e += blockDim.x) found |= k[head * key_blocks + e] < least_sum - share || v[head * key_blocks + e] == kBad;
    return found;
  }
};

// Products on pairs where that is faster.  Workgroups that meet a block that cannot be split leave their results to the kernels of attention.hip,
// which take the exponents that these return.
bool pair_suits(const Call &c, bool backward);
size_t pair_bytes(const Call &c, bool backward);  // of scratch
Exponents pair_forward(const Call &c, float *out, float *stat, const Pieces &pieces, int tiles, char *scratch, hipStream_t s);
// Where a backward pass writes: dq, or its pieces `row_stride` apart; dk and dv, or `parts` as dkv_kernel takes them.
struct Gradients {
  float *dq, *dk, *dv, *parts;
  int64_t row_stride;
  int row_pieces, pieces;
};
// Also what prepare_kernel writes to `rows`; dq (unless null), dk and dv (unless both are)
Exponents pair_backward(const Call &c, const float *out, const float *stat, const float *dout, Row *rows, const Gradients &to, int row_tiles, int key_tiles,
                        char *scratch, hipStream_t s);

}  // namespace attention
}  // namespace tf
