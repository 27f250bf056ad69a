// What the attention kernels share: the view of a call's arrays, which keys a query sees, and how a score comes out of a product.
//
//   s_ij = cap tanh(scale q_i k_j / cap) - slope |i + Tk - Tq - j|, seen keys only;   without a cap s = scale q k
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
  const float *spans;      // [queries, 2], of each batch entry where span_stride is not 0
  const float *slopes;     // of each query head
  int64_t span_stride;
  int batch, tq, tk, heads, key_heads, group, dim;
  int rows;                // tq * group: of a key head
  float scale, cap;        // cap 0: none
  bool causal;

  __device__ inline int64_t query_at(int b, int g, int r) const {  // of row r of key head g; also of o, do, dq
    return (((int64_t)b * tq + r / group) * heads + g * group + r % group) * dim;
  }
  __device__ inline int64_t key_at(int b, int g, int j) const { return (((int64_t)b * tk + j) * key_heads + g) * dim; }
  __device__ inline int64_t stat_at(int b, int g, int r) const { return ((int64_t)b * heads + g * group + r % group) * tq + r / group; }
  // The keys that query i sees: [lo, hi), lo >= hi for none.
  __device__ inline void seen(int b, int i, int &lo, int &hi) const {
    lo = 0;
    hi = tk;
    if (spans) {
      const float *span = spans + b * span_stride + 2 * (int64_t)i;
      const float first = span[0], last = span[1];
      // key j is seen where first <= j < last; a NaN sees none
      if (!(first < last)) hi = 0;
      else {
        if (first > 0.f) lo = first < (float)tk ? (int)ceilf(first) : tk;
        if (last < (float)tk) hi = last > 0.f ? (int)ceilf(last) : 0;
      }
    }
    if (causal) hi = min(hi, i + tk - tq + 1);
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

}  // namespace attention
}  // namespace tf
