// Gated feed-forward product, forward and backward (no counterpart in the reference).
//
//   g = x Wg, u = x Wu, h = act(g) u        x [M, K], Wg and Wu [K, F]
//   dg = dh u act'(g), du = dh act(g);  dx = dg Wg^T + du Wu^T,  dWg = x^T dg,  dWu = x^T du
//
// Large products run on fp16 pairs (gemm_pair.h), in three launches a pass (four for long maxima):
//
//   maxima   the largest magnitude of every row (and column) of the operands, by runs of them
//   split    every operand into its two fp16 numbers, in the order in which the products fetch them.  The gradients dg and du are
//            computed from g, u and dh on the way, in both launches, and never stored; they are split twice, by rows for dx and
//            by columns for dWg and dWu, because every sum needs a scale of its own for each of its operands
//   product  forward: the two weights' columns alternate in blocks of 32, so that a lane holds g and u of the same element and
//            the activation and the product of the two are the epilogue.  dx is one product over dg and du one behind the other, dWg
//            and dWu one of two halves, all in one launch.
//
// Little work is done in one launch from operands that stay in registers (namespace few).
#include "gemm_pair.h"
#include "gemm_split.h"
#include "internal.h"
#include "lanes.h"

#include <algorithm>
#include <cmath>

using namespace tf;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));
constexpr int kThreads = 256;

enum Activation { kSigmoid = 0, kRelu = 1, kSilu = 2, kGelu = 3, kGiven = -1 };

// Both from the hardware's exp2 and reciprocal, which are right to a step of the last place: what that leaves off is 2^-24 of
// the exponent's size, relative, on a value that gets small as the exponent grows; next to 1 it does not show.  The activations and
// their slopes are computed for every element of two passes, where expf and erff cost more than the loads.  Relative errors of sigmoid
// and SiLU: 2.4e-7 at -1, 1e-6 at -20, 4e-6 at -86, below which the reciprocal is subnormal and becomes zero.
__device__ inline float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g));
}
// Normal distribution function, and `bell` = exp(-g^2 / 2): the tail is t p(t) bell / 2 with t = 1 / (1 + |g| / sqrt 8) and p of six
// degrees, fitted to it so that the function is off by 7e-8 at most (evaluated in fp32 by 1.8e-7); relative to itself by 2e-6 down to -2,
// 5e-6 to -4, 3e-5 below.
__device__ inline float normal(float g, float &bell) {
  bell = __builtin_amdgcn_exp2f(-0.721347520444481704f * g * g);
  const float t = __builtin_amdgcn_rcpf(1.f + 0.353553390593273762f * __builtin_fabsf(g));
  float p = 0.5f * 0.0853855152f;
  p = p * t - 0.5f * 0.34268994f;
  p = p * t + 0.5f * 0.362460097f;
  p = p * t + 0.5f * 0.0629808057f;
  p = p * t + 0.5f * 0.269349229f;
  p = p * t + 0.5f * 0.280427633f;
  p = p * t + 0.5f * 0.282086729f;
  const float tail = p * t * bell;
  return g > 0.f ? 1.f - tail : tail;
}

// act(g) and act'(g)
template <int ACT>
__device__ inline void act_and_slope(float g, float &act, float &slope) {
  if (ACT == kRelu) {
    act = g > 0.f ? g : g != g ? g : 0.f;
    slope = g > 0.f ? 1.f : 0.f;
  } else if (ACT == kGelu) {
    float bell;
    const float cdf = normal(g, bell);
    act = g * cdf;
    slope = cdf + g * (0.39894228040143268f * bell);
  } else {
    const float s = sigmoid(g);
    act = ACT == kSigmoid ? s : g * s;
    slope = ACT == kSigmoid ? s * (1.f - s) : s * (1.f + g * (1.f - s));
  }
}
template <int ACT>
__device__ inline float act_of(float g) {
  float act, slope;
  act_and_slope<ACT>(g, act, slope);
  return act;
}

// Calls f with the activation as a compile-time constant.
template <class F>
void with_activation(int activation, F &&f) {
  switch (activation) {
    case kSigmoid: f(std::integral_constant<int, kSigmoid>{}); break;
    case kRelu: f(std::integral_constant<int, kRelu>{}); break;
    case kSilu: f(std::integral_constant<int, kSilu>{}); break;
    default: f(std::integral_constant<int, kGelu>{}); break;
  }
}

// Bound by HBM: 12 and 20 bytes an element.  4 096 x 4 096 28.6 us (7.0 TB/s, a part out of the last-level cache) and 59.0 (5.7), 64 x 4 096
// 3.6 and 3.8, a launch.
template <int ACT>
__global__ __launch_bounds__(kThreads) void activation_kernel(const float *g, const float *u, float *h, int64_t count) {
  const int64_t i = 4 * ((int64_t)blockIdx.x * kThreads + threadIdx.x);
  if (i + 4 <= count) {
    const f32x4 a = *reinterpret_cast<const f32x4u *>(g + i), b = *reinterpret_cast<const f32x4u *>(u + i);
    f32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = act_of<ACT>(a[j]) * b[j];
    *reinterpret_cast<f32x4u *>(h + i) = o;
  } else {
    for (int64_t j = i; j < count; ++j) h[j] = act_of<ACT>(g[j]) * u[j];
  }
}

template <int ACT>
__global__ __launch_bounds__(kThreads) void activation_backward_kernel(const float *g, const float *u, const float *dh,
                                                                      float *dg, float *du, int64_t count) {
  const int64_t i = 4 * ((int64_t)blockIdx.x * kThreads + threadIdx.x);
  float act, slope;
  if (i + 4 <= count) {
    const f32x4 a = *reinterpret_cast<const f32x4u *>(g + i), b = *reinterpret_cast<const f32x4u *>(u + i);
    const f32x4 d = *reinterpret_cast<const f32x4u *>(dh + i);
    f32x4 og, ou;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      act_and_slope<ACT>(a[j], act, slope);
      og[j] = d[j] * b[j] * slope;
      ou[j] = d[j] * act;
    }
    *reinterpret_cast<f32x4u *>(dg + i) = og;
    *reinterpret_cast<f32x4u *>(du + i) = ou;
  } else {
    for (int64_t j = i; j < count; ++j) {
      act_and_slope<ACT>(g[j], act, slope);
      const float d = dh[j], b = u[j];
      dg[j] = d * b * slope;
      du[j] = d * act;
    }
  }
}

// ---- operands of the large products ----------------------------------------------------------------------
using namespace tf::gemm;

// One or two matrices of one shape: weights, or the gradients of the projections, given or to be computed (dh).
struct Source {
  const float *p[2];
  const float *dh;   // not NULL: p are g and u, and the matrices are their gradients
  int rows, cols, activation;  // kGiven without dh

  template <int ACT>
  static __device__ inline void gradients(float g, float u, float d, float &dg, float &du) {
    float act, slope;
    act_and_slope<ACT>(g, act, slope);
    dg = d * u * slope;
    du = d * act;
  }
  __device__ inline float at(int which, int r, int c) const {
    if (r >= rows || c >= cols) return 0.f;
    const size_t i = (size_t)r * cols + c;
    if (!dh) return p[which][i];
    const float g = p[0][i], u = p[1][i], d = dh[i];
    float v[2];
    switch (activation) {
      case kSigmoid: gradients<kSigmoid>(g, u, d, v[0], v[1]); break;
      case kRelu: gradients<kRelu>(g, u, d, v[0], v[1]); break;
      case kSilu: gradients<kSilu>(g, u, d, v[0], v[1]); break;
      default: gradients<kGelu>(g, u, d, v[0], v[1]); break;
    }
    return v[which];
  }
  // four columns from c on of both matrices; zeros past the end.  ACT as `activation` says, kGiven: the matrices as they are
  template <int ACT>
  __device__ inline void four(int r, int c, f32x4 (&v)[2]) const {
    v[0] = v[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r >= rows || c >= cols) return;
    const size_t i = (size_t)r * cols + c;
    f32x4 d = v[0];
    if (c + 4 <= cols) {
      v[0] = *reinterpret_cast<const f32x4u *>(p[0] + i);
      if (ACT != kGiven || p[1]) v[1] = *reinterpret_cast<const f32x4u *>(p[1] + i);
      if (ACT != kGiven) d = *reinterpret_cast<const f32x4u *>(dh + i);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (c + e < cols) {
          v[0][e] = p[0][i + e];
          if (ACT != kGiven || p[1]) v[1][e] = p[1][i + e];
          if (ACT != kGiven) d[e] = dh[i + e];
        }
    }
    if constexpr (ACT != kGiven) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float dg, du;
        gradients<ACT>(v[0][e], v[1][e], d[e], dg, du);
        v[0][e] = dg;
        v[1][e] = du;
      }
    }
  }
};

// Calls f with the source's activation as a compile-time constant: one branch a workgroup, not one an element.
template <class F>
__device__ __forceinline__ void by_activation(const Source &src, F &&f) {
  switch (src.activation) {
    case kGiven: f(std::integral_constant<int, kGiven>{}); break;
    case kSigmoid: f(std::integral_constant<int, kSigmoid>{}); break;
    case kRelu: f(std::integral_constant<int, kRelu>{}); break;
    case kSilu: f(std::integral_constant<int, kSilu>{}); break;
    default: f(std::integral_constant<int, kGelu>{}); break;
  }
}

// What is made of a source.  By rows: both matrices behind each other along the reduction, `half_steps` steps each, a row's
// exponent common to both.  By columns: matrix w's block of 32 columns b is block b * col_mul + w * col_add.
// Maxima: [matrix][run of columns][row], [matrix][run of rows][column]; by rows the matrices' are one.
struct Job {
  Source src;
  int matrices;
  char *row_planes, *col_planes;  // NULL: not wanted
  int *row_exps, *col_exps;
  uint32_t *row_max, *col_max;
  int half_steps, col_steps, col_mul, col_add;
  bool col_wanted[2];
  int first_max, first_exps, first_split;  // the job's first workgroup of each launch
};
struct Jobs {
  Job job[3];
  int n;
  bool exps_apart;  // the exponents have a launch of their own
};

constexpr int kMaxRows = 64, kMaxCols = 128;   // a workgroup's part of the maxima
constexpr int kSplitTile = 64;                 // rows and columns of a workgroup's part of the split

__device__ inline uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// Bit patterns of magnitudes are in the order of the magnitudes, infinities and NaN above all.  Half a wave a row, all of a lane's
// loads under way at once.
__global__ __launch_bounds__(kThreads) void maxima_kernel(const Jobs jobs) {
  int n = jobs.n - 1;
  while (n > 0 && (int)blockIdx.x < jobs.job[n].first_max) --n;
  const Job &job = jobs.job[n];
  const int rows = job.src.rows, cols = job.src.cols, runs_c = (cols + kMaxCols - 1) / kMaxCols;
  const int run_c = ((int)blockIdx.x - job.first_max) % runs_c, run_r = ((int)blockIdx.x - job.first_max) / runs_c;
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const int c = run_c * kMaxCols + 4 * lane;
  __shared__ uint32_t of_groups[2][8][kMaxCols];
  uint32_t col[2][4] = {}, row[kMaxRows / 8];
  by_activation(job.src, [&](auto act) {
#pragma unroll
    for (int e = 0; e < kMaxRows / 8; ++e) {
      f32x4 v[2];
      job.src.four<decltype(act)::value>(run_r * kMaxRows + 8 * e + group, c, v);
      row[e] = 0;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t m = magnitude(v[w][i]);
          col[w][i] = max(col[w][i], m);
          row[e] = max(row[e], m);
        }
    }
  });
  if (job.row_planes) {
#pragma unroll
    for (int e = 0; e < kMaxRows / 8; ++e) {
      row[e] = lanes::largest<32>(row[e]);
      const int r = run_r * kMaxRows + 8 * e + group;
      if (lane == 0 && r < rows) job.row_max[(size_t)run_c * rows + r] = row[e];
    }
  }
  if (!job.col_planes) return;
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < 4; ++i) of_groups[w][group][4 * lane + i] = col[w][i];
  __syncthreads();
  const int w = threadIdx.x / kMaxCols, at = run_c * kMaxCols + (int)threadIdx.x % kMaxCols;
  if (at >= cols || w >= job.matrices) return;
  uint32_t m = 0;
#pragma unroll
  for (int g = 0; g < 8; ++g) m = max(m, of_groups[w][g][threadIdx.x % kMaxCols]);
  job.col_max[((size_t)w * ((rows + kMaxRows - 1) / kMaxRows) + run_r) * cols + at] = m;
}

// The power of two that brings the largest magnitude into [2^14, 2^15)
__device__ inline int exponent_of(uint32_t largest) {
  if (largest >= 0x7f800000u) return pair::kNotFinite;
  return largest == 0 ? 0 : 15 - __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, largest));
}

__device__ inline int finite(int exponent) { return exponent == pair::kNotFinite ? 0 : exponent; }
// the place of a column's exponent
__device__ inline int col_at(const Job &job, int w, int c) { return (c / 32 * job.col_mul + w * job.col_add) * 32 + c % 32; }

// The runs' maxima to exponents, those of 64 rows or columns a workgroup.  A launch of its own where there are kRunsApart runs and
// more, which every tile of the split would go through otherwise.  With it / without, us: backward of 1 024 x 4 096, 2 048 rows
// (32 runs) 284 / 284, 4 096 530 / 547, 16 384 1 884 / 2 113, 65 536 7 547 / 11 618; of 1 000 x 1 537, 777 rows 72 / 70, 4 096 212 /
// 214; forward of 512 x 1 376, 4 096 rows 60 / 56.
constexpr int kRunsApart = 64;
constexpr int kExpsThreads = 1024;
__global__ __launch_bounds__(kExpsThreads) void exponents_kernel(const Jobs jobs) {
  int n = jobs.n - 1;
  while (n > 0 && (int)blockIdx.x < jobs.job[n].first_exps) --n;
  const Job &job = jobs.job[n];
  const int rows = job.src.rows, cols = job.src.cols, of_rows = job.row_planes ? (rows + 63) / 64 : 0, of_cols = (cols + 63) / 64;
  const int group = (int)blockIdx.x - job.first_exps, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool by_rows = group < of_rows;
  const int w = by_rows ? 0 : (group - of_rows) / of_cols, at = (by_rows ? group : (group - of_rows) % of_cols) * 64 + lane;
  if (!by_rows && !job.col_wanted[w]) return;
  const int count = by_rows ? rows : cols;
  const int runs = by_rows ? (cols + kMaxCols - 1) / kMaxCols : (rows + kMaxRows - 1) / kMaxRows;
  const uint32_t *from = (by_rows ? job.row_max : job.col_max + (size_t)w * runs * cols) + min(at, count - 1);
  constexpr int WAVES = kExpsThreads / 64, LOADS = 4;
  uint32_t m = 0;
  for (int i = wave; i < runs; i += LOADS * WAVES) {
    uint32_t v[LOADS];  // a repeated value does not matter
#pragma unroll
    for (int e = 0; e < LOADS; ++e) v[e] = from[(size_t)min(i + e * WAVES, runs - 1) * count];
#pragma unroll
    for (int e = 0; e < LOADS; ++e) m = max(m, v[e]);
  }
  __shared__ uint32_t of_waves[WAVES][64];
  of_waves[wave][lane] = m;
  __syncthreads();
  if (wave > 0 || at >= (count + 31) / 32 * 32) return;
#pragma unroll
  for (int o = 1; o < WAVES; ++o) m = max(m, of_waves[o][lane]);
  const int exponent = at < count ? exponent_of(m) : 0;
  if (by_rows) job.row_exps[at] = exponent;
  else job.col_exps[col_at(job, w, at)] = exponent;
}

// Eight elements to the two halves of a lane's place in a fragment pair.
__device__ inline void split_eight(const float (&x)[8], int exponent, char *at) {
  pair::f16x8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = __builtin_ldexpf(x[i], exponent);
    h[i] = (_Float16)v;
    l[i] = (_Float16)((v - (float)h[i]) * pair::kLowScale);
  }
  *reinterpret_cast<pair::f16x8 *>(at) = h;
  *reinterpret_cast<pair::f16x8 *>(at + pair::kFragment) = l;
}

__global__ __launch_bounds__(kThreads) void split_kernel(const Jobs jobs) {
  constexpr int T = kSplitTile, LD = T + 4;
  int n = jobs.n - 1;
  while (n > 0 && (int)blockIdx.x < jobs.job[n].first_split) --n;
  const Job &job = jobs.job[n];
  const int rows = job.src.rows, cols = job.src.cols, tiles_c = (cols + T - 1) / T;
  const int r0 = ((int)blockIdx.x - job.first_split) / tiles_c * T, c0 = ((int)blockIdx.x - job.first_split) % tiles_c * T;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ __align__(16) float tile[2][T][LD];
  __shared__ int row_exp[T], col_exp[2][T];

  // the tile, 16 lanes a row
  by_activation(job.src, [&](auto act) {
#pragma unroll
    for (int e = 0; e < T / 16; ++e) {
      const int r = e * 16 + tid / 16, c = tid % 16 * 4;
      f32x4 v[2];
      job.src.four<decltype(act)::value>(r0 + r, c0 + c, v);
      *reinterpret_cast<f32x4 *>(&tile[0][r][c]) = v[0];
      if (job.matrices > 1) *reinterpret_cast<f32x4 *>(&tile[1][r][c]) = v[1];
    }
  });
  if (jobs.exps_apart) {
    if (tid < T) {
      if (job.row_planes) row_exp[tid] = finite(job.row_exps[min(r0 + tid, rows - 1)]);
      if (job.col_planes)
        for (int w = 0; w < job.matrices; ++w)
          if (job.col_wanted[w]) col_exp[w][tid] = finite(job.col_exps[col_at(job, w, min(c0 + tid, cols - 1))]);
    }
  } else {  // four lanes each; the tiles at the reduction's beginning write them down
    const int of = tid / 4, part = tid % 4;
    auto largest = [&](const uint32_t *from, int runs, int64_t stride) {
      uint32_t m = 0;
      for (int i = part; i < runs; i += 16) {
        uint32_t v[4];  // a repeated value does not matter
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from[min(i + 4 * e, runs - 1) * stride];
        m = max(m, max(max(v[0], v[1]), max(v[2], v[3])));
      }
      m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
      return max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
    };
    if (job.row_planes) {
      const int r = r0 + of;
      const int e = exponent_of(largest(job.row_max + min(r, rows - 1), (cols + kMaxCols - 1) / kMaxCols, rows));
      if (part == 0) {
        row_exp[of] = finite(e);
        if (c0 == 0 && r < (rows + 31) / 32 * 32) job.row_exps[r] = r < rows ? e : 0;
      }
    }
    if (job.col_planes) {
      const int runs = (rows + kMaxRows - 1) / kMaxRows, c = c0 + of;
      for (int w = 0; w < job.matrices; ++w) {
        if (!job.col_wanted[w]) continue;
        const int e = exponent_of(largest(job.col_max + (size_t)w * runs * cols + min(c, cols - 1), runs, cols));
        if (part == 0) {
          col_exp[w][of] = finite(e);
          if (r0 == 0 && c < (cols + 31) / 32 * 32) job.col_exps[col_at(job, w, c)] = c < cols ? e : 0;
        }
      }
    }
  }
  __syncthreads();
  const int along = lane & 31, eight = lane >> 5 << 3;  // a lane's row and its elements in a fragment
  for (int w = 0; w < job.matrices; ++w)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int b = (wave + 4 * i) >> 2, step = wave & 3;
      float x[8];
      if (job.row_planes && r0 / 32 + b < (rows + 31) / 32 && c0 / 16 + step < job.half_steps) {
        const float *from = &tile[w][b * 32 + along][step * 16 + eight];
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          const f32x4 v = *reinterpret_cast<const f32x4 *>(from + k);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[k + j] = v[j];
        }
        const size_t at = (size_t)(r0 / 32 + b) * (job.matrices * job.half_steps) + w * job.half_steps + c0 / 16 + step;
        split_eight(x, row_exp[b * 32 + along], job.row_planes + at * pair::kStepBytes + lane * 16);
      }
      if (job.col_planes && job.col_wanted[w] && c0 / 32 + b < (cols + 31) / 32 && r0 / 16 + step < job.col_steps) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = tile[w][step * 16 + eight + k][b * 32 + along];
        const size_t at = (size_t)((c0 / 32 + b) * job.col_mul + w * job.col_add) * job.col_steps + r0 / 16 + step;
        split_eight(x, col_exp[w][b * 32 + along], job.col_planes + at * pair::kStepBytes + lane * 16);
      }
    }
}

// ---- the products' ends ------------------------------------------------------------------------------------
// Stores past the last row fall behind the buffer, those past the last column are sent there.  They go past the caches, which hold
// the operands: 4 096 x 1 024 x 4 096 forward 227 -> 216 us, the sublayer that reads h next 277 -> 276.
__device__ inline void store_past(__amdgpu_buffer_rsrc_t r, uint32_t byte_off, float v) {
  constexpr int NT = 2;  // in the cache-policy operand
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, v), r, (int)byte_off, 0, NT);
}
struct Rows {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ inline Rows(float *out, int m0, int rows, int cols)
      : rsrc(make_rsrc(out ? out + (size_t)m0 * cols : nullptr, out ? (uint32_t)min(rows - m0, pair::BM) * (uint32_t)cols * 4u : 0u)) {}
};

// h = act(g) u from the two columns that a lane holds, and g and u themselves where pre is wanted
template <int ACT>
struct StoreGated {
  float *g, *u, *h;  // NULL: not wanted
  int rows, cols;
  struct State {
    Rows g, u, h;
  };
  __device__ inline State begin(int m0, int) const { return {Rows(g, m0, rows, cols), Rows(u, m0, rows, cols), Rows(h, m0, rows, cols)}; }
  template <int TN>
  __device__ inline void store(const State &s, int m, int block, int lcol, const float (&v)[TN]) const {
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      const int f = (block + j) / 2 * 32 + lcol;
      const uint32_t off = f < cols ? ((uint32_t)m * (uint32_t)cols + (uint32_t)f) * 4u : OOB;
      if (g) {  // uniform
        store_past(s.g.rsrc, off, v[j]);
        store_past(s.u.rsrc, off, v[j + 1]);
      }
      if (h) store_past(s.h.rsrc, off, act_of<ACT>(v[j]) * v[j + 1]);
    }
  }
};
struct StoreHalves {
  float *out[2];
  int rows, cols;
  using State = Rows;
  __device__ inline State begin(int m0, int half) const { return Rows(half ? out[1] : out[0], m0, rows, cols); }
  template <int TN>
  __device__ inline void store(const State &s, int m, int block, int lcol, const float (&v)[TN]) const {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = (block + j) * 32 + lcol;
      store_past(s.rsrc, n < cols ? ((uint32_t)m * (uint32_t)cols + (uint32_t)n) * 4u : OOB, v[j]);
    }
  }
};

// Operands as they were, for tiles with rows that are not finite
struct OfRows {  // of a matrix, or of two behind each other along the reduction, half_k elements each
  static constexpr bool kAlongRows = false;
  Source src;
  int half_k;
  __device__ inline float operator()(int row, int k) const { return k < half_k ? src.at(0, row, k) : src.at(1, row, k - half_k); }
};
struct OfColumnsInTurn {  // of two, in blocks of 32
  static constexpr bool kAlongRows = true;
  Source src;
  __device__ inline float operator()(int, int row, int k) const { return src.at(row / 32 % 2, k, row / 64 * 32 + row % 32); }
};
struct OfEither {  // of a backward product: dx by rows, the weights' gradients by columns
  static constexpr bool kAlongRows = false;
  OfRows rows;
  bool columns;
  __device__ inline float operator()(int row, int k) const { return (*this)(0, row, k); }
  __device__ inline float operator()(int half, int row, int k) const { return columns ? rows.src.at(half, k, row) : rows(row, k); }
};
template <int ACT>
struct Forward {
  static constexpr int kCount = 1;
  pair::Product<StoreGated<ACT>, OfRows, OfColumnsInTurn> p[1];
};
struct Backward {
  static constexpr int kCount = 2;
  pair::Product<StoreHalves, OfEither, OfEither> p[2];  // without a workgroup where it is not wanted
};

int steps_of(int k) { return cdiv(k, 32) * 2; }  // an even number

// Scratch of a call, laid out before it is had.
struct Layout {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};
struct PackedAt {
  size_t planes, exps;
  int blocks, steps;
  PackedAt() = default;
  PackedAt(Layout &l, int blocks_, int steps_, int operands = 1)
      : planes(l.take((size_t)operands * blocks_ * steps_ * pair::kStepBytes)), exps(l.take((size_t)operands * blocks_ * 32 * 4)),
        blocks(blocks_), steps(steps_) {}
  pair::Packed in(char *base) const { return {base + planes, (const int *)(base + exps), blocks, steps}; }
};

// Tiles of a product.
pair::Work tiles_of(int m_blocks, int n_blocks, int halves) {
  const int tile = pair::BM / 32;
  pair::Work w{};
  w.tiles_m = cdiv(m_blocks, tile);
  w.half_tiles = cdiv(n_blocks, tile);
  w.tiles_n = w.half_tiles * halves;
  return w;
}
// Pieces of a launch's one or two products, those that take the least time by a model: a step takes a workgroup that has its CU for itself 0.4 us
// and two that share one 0.65, a launch of more than two workgroups a CU ends with a part of them idle, and every piece writes its
// tile, all of which one workgroup reads, 6 us for a CU's piece times the pieces.  Over 110 sizes of both passes what it picks takes 0.6 per cent longer than the
// fastest that there is; pieces of as many steps as a CU has in all, four at most, 3.0.  us in 1 x 1 / picked: backward of
// 1 024 x 4 096, 777 rows 187 / 133, 4 096 rows 528 / 501; of 2 048 x 8 192, 777 rows 511 / 429; forward of 4 096 x 1 024, 512 rows
// 94 / 66.
constexpr int kMaxPieces = 8, kLeastSteps = 12;
struct Extent {
  int tiles, steps, pieces;  // no tiles: not there
  int steps_a_piece() const { return cdiv(steps / 2, pieces) * 2; }
};
double cost(const Extent (&e)[2]) {
  const double alone = 0.4, shared = 0.326, cus = num_cus();
  double groups = 0, work = 0, longest = 0, shortest = 1e30, folds = 0, last = 0;
  for (const Extent &x : e) {
    if (x.tiles == 0) continue;
    const double n = (double)x.tiles * x.pieces;
    last = x.steps_a_piece();
    groups += n;
    work += n * last;
    longest = std::max(longest, last);
    shortest = std::min(shortest, last);
    if (x.pieces > 1) folds += 6.0 * n * x.pieces / cus + 2.0;
  }
  if (groups <= cus) return longest * alone + folds;
  double time = std::max(work / cus * shared, longest * alone);
  const double idle = std::fmod(groups, 2 * cus) / (2 * cus);
  if (groups <= 2 * cus) time = std::max(time, 2 * shared * shortest + alone * (longest - shortest));
  else if (idle > 0) time = std::max(time, work / cus * shared + last * shared * (1 - idle));
  return time + folds;
}
void choose_pieces(Extent (&e)[2]) {
  Extent trial[2] = {e[0], e[1]};
  auto most = [](const Extent &x) {  // a ticket a tile
    return x.tiles == 0 || x.tiles > kFoldTicketSlots / 2 ? 1 : std::max(1, std::min(kMaxPieces, x.steps / kLeastSteps));
  };
  double least = 1e30;
  for (trial[0].pieces = 1; trial[0].pieces <= most(e[0]); ++trial[0].pieces)
    for (trial[1].pieces = 1; trial[1].pieces <= most(e[1]); ++trial[1].pieces) {
      const double c = cost(trial);
      if (c >= least) continue;
      least = c;
      e[0] = trial[0];
      e[1] = trial[1];
    }
}
// Its scratch's place, where there are several
size_t cut(Layout &l, pair::Work &w, const Extent &e) {
  w.steps_per_piece = e.steps_a_piece();
  w.pieces = cdiv(e.steps, w.steps_per_piece);
  return w.pieces > 1 ? l.take((size_t)e.tiles * w.pieces * pair::BM * pair::BN * 4) : 0;
}
// `tickets`: one for each of its tiles
void give(pair::Work &w, char *base, size_t scratch, unsigned *tickets) {
  if (w.pieces < 2) return;
  w.scratch = (float *)(base + scratch);
  w.tickets = tickets;
}

// The two launches in front of the products, three for long maxima.
struct Splitting {
  Jobs jobs{};
  int maxima_groups = 0, exps_groups = 0, split_groups = 0;
  size_t row_max[3], col_max[3];
  void add(Layout &l, const Source &src, int matrices, bool by_rows, bool by_columns) {
    Job &j = jobs.job[jobs.n];
    j.src = src;
    j.matrices = matrices;
    const int runs_c = cdiv(src.cols, kMaxCols), runs_r = cdiv(src.rows, kMaxRows);
    row_max[jobs.n] = by_rows ? l.take((size_t)runs_c * src.rows * 4) : 0;
    col_max[jobs.n] = by_columns ? l.take((size_t)matrices * runs_r * src.cols * 4) : 0;
    j.half_steps = steps_of(src.cols);
    j.col_steps = steps_of(src.rows);
    j.col_mul = 1;
    j.col_add = cdiv(src.cols, 32);
    j.col_wanted[0] = j.col_wanted[1] = true;
    j.first_max = maxima_groups;
    j.first_exps = exps_groups;
    j.first_split = split_groups;
    maxima_groups += runs_c * runs_r;
    exps_groups += (by_rows ? cdiv(src.rows, 64) : 0) + (by_columns ? matrices * cdiv(src.cols, 64) : 0);
    jobs.exps_apart |= (by_rows && runs_c >= kRunsApart) || (by_columns && runs_r >= kRunsApart);
    split_groups += cdiv(src.rows, kSplitTile) * cdiv(src.cols, kSplitTile);
    ++jobs.n;
  }
  void rows_to(int n, const PackedAt &p, char *base) {
    jobs.job[n].row_planes = base + p.planes;
    jobs.job[n].row_exps = (int *)(base + p.exps);
    jobs.job[n].row_max = (uint32_t *)(base + row_max[n]);
  }
  void columns_to(int n, const PackedAt &p, char *base) {
    jobs.job[n].col_planes = base + p.planes;
    jobs.job[n].col_exps = (int *)(base + p.exps);
    jobs.job[n].col_max = (uint32_t *)(base + col_max[n]);
  }
  void launch(hipStream_t s) const {
    hipLaunchKernelGGL(maxima_kernel, dim3((unsigned)maxima_groups), dim3(kThreads), 0, s, jobs);
    if (jobs.exps_apart)
      hipLaunchKernelGGL(exponents_kernel, dim3((unsigned)exps_groups), dim3(kExpsThreads), 0, s, jobs);
    hipLaunchKernelGGL(split_kernel, dim3((unsigned)split_groups), dim3(kThreads), 0, s, jobs);
  }
};

// Rows of a workgroup where few are: 64 once that fills half of the CUs.  32 / 64, us: 192 rows of 1 000 x 2 731 (129 workgroups of 64) 38.6 /
// 30.7, 64 of 4 096 x 11 008 (172) 156 / 110, 256 of 1 024 x 4 096 (256) 36.1 / 34.2; 128 of 1 024 x 4 096 (128) 21.3 / 25.1, 64 of
// 1 000 x 2 731 (43) 18.0 / 21.0.
namespace few {
constexpr int C = 2, kCols = 32 * C;  // columns of a lane, of a workgroup
int rows_of(int64_t M, int64_t F) { return (int64_t)cdiv(F, kCols) * cdiv(M, 64) > num_cus() / 2 ? 64 : 32; }
}  // namespace few

// Whether the environment asks for the fp32 instruction, as it may of every other contraction: TINYFLOW_SPLIT=0.  Then all products are
// those of namespace few, whose runs go the way of runs that cannot be sliced.
bool on_fp32() {
  const char *e = getenv("TINYFLOW_SPLIT");
  return e && *e && atoi(e) == 0;
}

// Whether the forward pass runs on pairs, or in registers with nothing stored split (namespace few): us, fitted.  K x F, rows, few
// / pairs: 1 024 x 4 096, 128 22 / 43, 256 34 / 46, 320 61 / 49, 512 68 / 53; 2 048 x 8 192, 128 63 / 132, 192 114 / 133, 256 123 /
// 135, 320 168 / 159; 4 096 x 11 008, 192 301 / 363, 320 445 / 433, 512 680 / 453; 1 000 x 2 731, 320 35 / 46, 384 64 / 45; 512 x
// 1 376, 512 21 / 29, 768 41 / 31; 256 x 1 024, 1 024 17 / 24.
bool forward_on_pairs(int64_t M, int64_t K, int64_t F) {
  if (K >= 1 << 22 || F >= 1 << 22 || on_fp32()) return false;  // a tile's rows would pass a buffer's end
  const int rows = few::rows_of(M, F);
  const double few = 12.0 + 4.0 * cdiv(M, rows) * rows * (double)K * cdiv(F, few::kCols) * few::kCols / 110e6;
  const double m = (double)cdiv(M, 32) * 32, k = (double)cdiv(K, 32) * 32, f = (double)cdiv(F, 32) * 32;
  const double pairs = 20.0 + (24.0 * k * f + 12.0 * m * k) / 4.8e6 + 4.0 * m * k * f / 380e6;
  return pairs < few;
}
// The backward pass likewise.  K x F, rows, few / pairs: 128 x 512, 1 024 20 / 35; 256 x 1 024, 1 024 36 / 40; 512 x 1 376, 64 17 / 38, 384 38 /
// 41, 512 48 / 41; 1 000 x 1 537 (rows that start inside a line), 64 23 / 41, 128 37 / 43, 192 52 / 46; 2 083 x 6 733, 57 178 / 147; 1 024 x 4 096, 24 28 / 54, 128 55 /
// 65, 192 76 / 71, 512 171 / 96; 2 048 x 8 192, 24 78 / 152, 64 120 / 168, 96 167 / 182, 128 198 / 187.  Long reductions into few tiles:
// 1 x 7, 524 288 389 / 1 264; 16 x 16, 1 048 576 758 / 2 543; 64 x 64, 16 384 33 / 64, 65 536 91 / 184; 128 x 256, 65 536 240 / 382; 256 x 512,
// 16 384 210 / 146, 65 536 851 / 565; 128 x 512, 8 192 61 / 67; 128 x 65 536, 512 492 / 722; 512 x 16 384, 512 401 / 241.  That also keeps
// pairs from narrow extents, which their blocks of 32 hold several times over (2^26 rows of 1 x 7: 43 GB beside arrays of 6).
bool backward_on_pairs(int64_t M, int64_t K, int64_t F) {
  if (M == 0 || K == 0 || F == 0 || K >= 1 << 22 || F >= 1 << 22 || on_fp32()) return false;
  const double m = (double)cdiv(M, 32) * 32, k = (double)cdiv(K, 64) * 64, f = (double)cdiv(F, 32) * 32;
  const double few = 11.0 + 1.3e-6 * k * f + (F % 32 ? 150e-9 : 88e-9) * m * k * f;
  // a piece of the longest reduction, one step behind the other: few tiles leave CUs idle
  const double alone = 0.34 * std::max(steps_of((int)M), 2 * steps_of((int)F)) / kMaxPieces;
  const double pairs = 30.0 + 6.5e-6 * k * f + 0.59e-6 * m * (k + 3 * f) + std::max(18.8e-9 * m * k * f, alone);
  return pairs < few;
}

// Scratch goes back to the pool when a call returns; a graph would go on using it.
constexpr int64_t kCaptured = -1;

// These return 0, the bytes of scratch that could not be had, or kCaptured.
int64_t forward_by_pairs(int M, int K, int F, const float *x, const float *gate, const float *up, float *pre, float *h, int activation,
                         hipStream_t s) {
  Layout l;
  Splitting split;
  const Source xs{{x, nullptr}, nullptr, M, K, kGiven}, ws{{gate, up}, nullptr, K, F, kGiven};
  split.add(l, xs, 1, true, false);
  split.add(l, ws, 2, false, true);
  const int f_blocks = cdiv(F, 32);
  const PackedAt a(l, cdiv(M, 32), steps_of(K)), b(l, 2 * f_blocks, steps_of(K));
  pair::Work work = tiles_of(a.blocks, b.blocks, 1);
  Extent pieces[2] = {{work.tiles_m * work.tiles_n, a.steps, 1}, {0, 0, 1}};
  choose_pieces(pieces);
  const size_t scratch = cut(l, work, pieces[0]);
  if (being_captured(s)) return kCaptured;
  unsigned *tickets = fold_tickets(s);
  char *base = tickets ? (char *)device_alloc(l.bytes, s) : nullptr;
  if (!base) return (int64_t)block_bytes(l.bytes);
  split.rows_to(0, a, base);
  split.columns_to(1, b, base);
  split.jobs.job[1].col_mul = 2;
  split.jobs.job[1].col_add = 1;
  split.launch(s);
  give(work, base, scratch, tickets);
  with_activation(activation, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    const Forward<ACT> product{{{a.in(base), b.in(base), work, StoreGated<ACT>{pre, pre ? pre + (size_t)M * F : nullptr, h, M, F},
                                 OfRows{xs, a.steps * pair::BK}, OfColumnsInTurn{ws}}}};
    hipLaunchKernelGGL(pair::gemm_kernel<Forward<ACT>>, dim3((unsigned)product.p[0].groups()), dim3(THREADS), 0, s, product);
  });
  device_free(base, s);
  return 0;
}

int64_t backward_by_pairs(int M, int K, int F, const float *x, const float *gate, const float *up, const Source &d, float *dx,
                          float *dgate, float *dup, hipStream_t s) {
  Layout l;
  Splitting split;
  const Source xs{{x, nullptr}, nullptr, M, K, kGiven}, ws{{gate, up}, nullptr, K, F, kGiven};
  const bool weights = dgate || dup;
  PackedAt d_rows, w_rows, d_cols, x_cols;
  pair::Work to_x{}, to_w{};
  split.add(l, d, 2, dx != nullptr, weights);
  if (dx) split.add(l, ws, 2, true, false);
  if (weights) split.add(l, xs, 1, false, true);
  const int f_blocks = cdiv(F, 32), k_blocks = cdiv(K, 32), m_blocks = cdiv(M, 32);
  if (dx) {
    d_rows = PackedAt(l, m_blocks, 2 * steps_of(F));
    w_rows = PackedAt(l, k_blocks, 2 * steps_of(F));
    to_x = tiles_of(m_blocks, k_blocks, 1);
  }
  if (weights) {
    d_cols = PackedAt(l, f_blocks, steps_of(M), 2);
    x_cols = PackedAt(l, k_blocks, steps_of(M));
    to_w = tiles_of(k_blocks, f_blocks, 2);
  }
  // pieces as for all three gradients, so that each has the same bits alone
  const pair::Work all_x = tiles_of(m_blocks, k_blocks, 1), all_w = tiles_of(k_blocks, f_blocks, 2);
  Extent pieces[2] = {{all_x.tiles_m * all_x.tiles_n, 2 * steps_of(F), 1}, {all_w.tiles_m * all_w.tiles_n, steps_of(M), 1}};
  choose_pieces(pieces);
  const size_t x_scratch = dx ? cut(l, to_x, pieces[0]) : 0, w_scratch = weights ? cut(l, to_w, pieces[1]) : 0;
  if (weights && (!dgate || !dup)) {
    to_w.tiles_n = to_w.half_tiles;
    to_w.first_half = dgate ? 0 : 1;
  }
  unsigned *tickets = fold_tickets(s);
  char *base = tickets ? (char *)device_alloc(l.bytes, s) : nullptr;
  if (!base) return (int64_t)block_bytes(l.bytes);
  if (dx) {
    split.rows_to(0, d_rows, base);
    split.rows_to(1, w_rows, base);
  }
  if (weights) {
    split.columns_to(0, d_cols, base);
    split.jobs.job[0].col_wanted[0] = dgate != nullptr;
    split.jobs.job[0].col_wanted[1] = dup != nullptr;
    split.columns_to(dx ? 2 : 1, x_cols, base);
  }
  split.launch(s);
  give(to_x, base, x_scratch, tickets);
  give(to_w, base, w_scratch, tickets + kFoldTicketSlots / 2);
  Backward products{};
  if (dx)
    products.p[0] = {d_rows.in(base), w_rows.in(base), to_x, StoreHalves{{dx, nullptr}, M, K},
                     {{d, steps_of(F) * pair::BK}, false}, {{ws, steps_of(F) * pair::BK}, false}};
  if (weights)
    products.p[1] = {x_cols.in(base), d_cols.in(base), to_w, StoreHalves{{dgate, dup}, K, F}, {{xs, 0}, true}, {{d, 0}, true}};
  hipLaunchKernelGGL(pair::gemm_kernel<Backward>, dim3((unsigned)(products.p[0].groups() + products.p[1].groups())), dim3(THREADS),
                     0, s, products);
  device_free(base, s);
  return 0;
}

// ---- little work: nothing stored split ---------------------------------------------------------------------------
// Both projections, the activation and the product for 32 or 64 rows a workgroup: nothing is staged.  A wave owns 32 C columns of both
// weights and a run of the reduction; the C columns of a lane's load belong to C matrix instructions (columns C (lane mod 32) + j of
// the j-th), so that the lanes' order costs nothing.  In a group of sixteen reduction elements lanes 0..31 hold the first eight and
// lanes 32..63 the others, which is the operand of one bf16 instruction: the values are split in registers into three slices each
// (gemm_split.h), six products of a weight's slices serve each 32 rows.  DEPTH groups are under way.  The waves of a workgroup have
// runs of their own, added through LDS, and several workgroups more of them, added by the last one to finish (gemm_core.h: Fold), in
// their order.  A run whose sums are not finite is computed again with the fp32 instruction.
//
// Bound by the weights' bytes for few rows, by the splitting (five and a half vector instructions a value) for more: with the fp32
// instruction / so, us, rows of K x F: 24 of 1 000 x 2 731 14.5 / 12.5, of 2 048 x 8 192 36.5 / 31.5 (4.3 TB/s), of 4 096 x 11 008 102 / 85;
// 128 of 1 024 x 4 096 26.2 / 21.3, of 2 048 x 8 192 86 / 63 (138 TFLOP/s); 256 of 1 000 x 2 731 47 / 32.  The loads' order matters as
// much: where the compiler waits for both groups at once, 5 to 15 per cent.  Three groups under way need the registers of the second sums.
namespace few {
constexpr int kWaves = 4, kDepth = 2, kGroup = 16;
typedef float Columns __attribute__((ext_vector_type(C)));
typedef Columns ColumnsU __attribute__((aligned(4)));

struct Args {
  const float *x, *gate, *up;
  float *g, *u, *h;  // NULL: not wanted
  int M, K, F, strips, k_per_group, pieces;
  bool alone;        // every wave has a strip for itself, a workgroup four side by side
  bool exact;        // with the fp32 instruction from the start,
  int skipped;       // the loop on slices left out: K then, else 0.  Two words: one would live through the loop, in a register that it needs
  float *scratch;    // [strip][row group][piece][accumulator][g, u][lane][C]
  unsigned *tickets;
};

template <int N, int POLICY>
__device__ inline auto load_columns(__amdgpu_buffer_rsrc_t r, uint32_t byte_off, int uniform_off = 0) {
  typedef float V __attribute__((ext_vector_type(N)));
  if constexpr (N == 4) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, (int)byte_off, uniform_off, POLICY));
  else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, (int)byte_off, uniform_off, POLICY));
}
template <int POLICY, class V>
__device__ inline void store_columns(__amdgpu_buffer_rsrc_t r, uint32_t byte_off, const V &v) {
  if constexpr (sizeof(V) == 16)
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(__attribute__((__vector_size__(16))) unsigned, v), r, (int)byte_off, 0, POLICY);
  else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(__attribute__((__vector_size__(8))) unsigned, v), r, (int)byte_off, 0, POLICY);
}

// Whether neighbouring strips share an XCD: where they share lines, because the weights' rows start inside one.  Spread / so, us: one row of
// 1 000 x 2 731 8.6 / 7.8, 64 rows 18.0 / 15.9, 128 rows 23.6 / 21.1; of 1 024 x 4 096 8.3 / 8.6, 16.3 / 16.4, 21.8 / 22.2, one row of
// 2 048 x 8 192 27.4 / 29.6.
__device__ inline bool by_neighbours(int F) { return F % 32 != 0; }

// The three slices of eight reduction elements, as an operand.
struct Slices {
  split::bf16x8 of[3];
  template <class Get>
  __device__ inline explicit Slices(Get &&get) {
    uint32_t words[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t pair_of[3];
      split::split_pair(get(2 * i), get(2 * i + 1), pair_of);
#pragma unroll
      for (int q = 0; q < 3; ++q) words[q][i] = pair_of[q];
    }
#pragma unroll
    for (int q = 0; q < 3; ++q)
      of[q] = __builtin_bit_cast(split::bf16x8, split::u32x4v{words[q][0], words[q][1], words[q][2], words[q][3]});
  }
};

// BLOCKS blocks of 32 rows
template <int ACT, int BLOCKS>
__global__ __launch_bounds__(kThreads, BLOCKS == 1 ? 2 : 1) void forward_kernel(const Args a) {
  constexpr int kRows = 32 * BLOCKS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, along = lane & 31;
  const int groups = gridDim.x, id = blockIdx.y * groups + blockIdx.x;
  const int logical = by_neighbours(a.F) ? xcd_contiguous(id, groups * gridDim.y) : id;
  const int across = a.alone ? (a.strips + kWaves - 1) / kWaves : a.strips;
  const int piece = logical / groups, group = logical % groups, row_groups = groups / across;
  const int strip = (by_neighbours(a.F) ? group / row_groups : group % across) * (a.alone ? kWaves : 1) + (a.alone ? wave : 0);
  const int m0 = (by_neighbours(a.F) ? group % row_groups : group / across) * kRows;
  const int rows = min(kRows, a.M - m0), c0 = strip * kCols;
  const int of_wave = a.alone ? a.k_per_group : a.k_per_group / kWaves;
  const int k_begin = a.alone ? 0 : piece * a.k_per_group + wave * of_wave, k_end = min(a.K, k_begin + of_wave);
  // Wave q adds up accumulators OWN q .. OWN q + OWN - 1, ROUND waves at a time; accumulator v of a block holds rows 8 (v / 4) + 4 half
  // + v mod 4.
  constexpr int OWN = 16 * BLOCKS / kWaves, ROUND = kWaves / 2;
  __shared__ Columns part[ROUND][kWaves - 1][OWN][2][64];  // [wave that adds][wave that has][accumulator][g, u][lane]
  __shared__ unsigned last;

  const uint32_t bytes = (uint32_t)k_end * (uint32_t)a.F * 4u;  // nothing behind the run is fetched
  const __amdgpu_buffer_rsrc_t rsrc[2] = {make_rsrc(a.gate, bytes), make_rsrc(a.up, bytes)};
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, (uint32_t)a.M * (uint32_t)a.K * 4u);
  // a lane's columns past the end may hold the next row's values: they are not stored
  const int c = c0 + C * along;
  const uint32_t col_off = c < a.F ? (uint32_t)c * 4u : OOB;
  uint32_t row_off[BLOCKS];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i)
    row_off[i] = 32 * i + along < rows ? (uint32_t)(m0 + 32 * i + along) * (uint32_t)a.K * 4u : OOB;

  f32x16 acc[2][C][BLOCKS], low[2][C][BLOCKS];  // products of the two highest slices, and of others
  auto clear = [&](f32x16 (&sums)[2][C][BLOCKS]) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) sums[w][j][i][v] = 0.f;
  };
  clear(acc);
  clear(low);

  // COUNT reduction elements of a lane, those of the upper half of the wave COUNT further on: of x, of one row a block; of the weights,
  // of C columns.  Behind the run's end they hold what there is, of the weights zeros and the last row again: x counts as zero there, from
  // `valid` of a lane's on, once it is used.  The uniform part of an address is a scalar, inside the buffer.
  const uint32_t row_bytes = (uint32_t)a.F * 4u;
  const int k_last = max(k_end - 1, 0);
  auto load_x = [&](int k0, auto &to) {
    constexpr int COUNT = sizeof(to[0]) / sizeof(float);
    const int from = min(k0, k_last) * 4;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
      for (int s = 0; s < COUNT; s += 4) {
        const f32x4v v = __builtin_bit_cast(
            f32x4v, __builtin_amdgcn_raw_buffer_load_b128(xr, (int)(row_off[i] + (uint32_t)(COUNT * half + s) * 4u), from, 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) to[i][s + e] = v[e];
      }
  };
  auto load_weights = [&](int k0, auto &to) {
    constexpr int COUNT = sizeof(to[0]) / sizeof(Columns);
    const uint32_t lane_off = col_off + (uint32_t)(COUNT * half) * row_bytes;
#pragma unroll
    for (int s = 0; s < COUNT; ++s) {
      const int from = (int)((uint32_t)min(k0 + s, k_last) * row_bytes);
#pragma unroll
      for (int w = 0; w < 2; ++w) to[w][s] = load_columns<C, 0>(rsrc[w], lane_off, from);
    }
  };
  float xv[kDepth][BLOCKS][8];
  Columns wv[kDepth][2][8];
  auto load = [&](int at, int k0) {
    load_x(k0, xv[at]);
    load_weights(k0, wv[at]);
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    load(d, k_begin + kGroup * d);
    __builtin_amdgcn_sched_barrier(0);  // in the order of the loop: the wait for one group leaves the others under way
  }
  for (int k0 = k_begin + a.skipped; k0 < k_end; k0 += kGroup * kDepth)
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int valid = k_end - (k0 + kGroup * d) - 8 * half;
      split::bf16x8 xs[BLOCKS][3];
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) {
        const Slices slices([&](int k) { return k < valid ? xv[d][i][k] : 0.f; });
#pragma unroll
        for (int q = 0; q < 3; ++q) xs[i][q] = slices.of[q];
      }
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const Slices weights([&](int k) { return wv[d][w][k][j]; });
#pragma unroll
          for (int p = 0; p < 6; ++p) {
            constexpr int of_x[6] = {0, 0, 1, 0, 1, 2}, of_w[6] = {0, 1, 0, 2, 1, 0};
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) {
              f32x16 &sum = p == 0 ? acc[w][j][i] : low[w][j][i];
              sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xs[i][of_x[p]], weights.of[of_w[p]], sum, 0, 0, 0);
            }
          }
        }
      load(d, k0 + kGroup * (d + kDepth));
      __builtin_amdgcn_sched_barrier(0);  // nothing of the next group, whose loads may still be under way, in front of this one
    }
  float finite = 0.f;
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          acc[w][j][i][v] = (acc[w][j][i][v] + low[w][j][i][v]) * split::kUnscale;
          finite = __builtin_fmaf(acc[w][j][i][v], 0.f, finite);  // NaN of an infinity or a NaN
        }
  if (a.exact || __any(finite != finite)) {
    clear(acc);
#pragma unroll 1
    for (int k0 = k_begin; k0 < k_end; k0 += 8) {
      float x4[BLOCKS][4];
      Columns w4[2][4];
      load_weights(k0, w4);
      load_x(k0, x4);
      const int valid = k_end - k0 - 4 * half;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int j = 0; j < C; ++j)
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i)
              acc[w][j][i] = __builtin_amdgcn_mfma_f32_32x32x2f32(s < valid ? x4[i][s] : 0.f, s < valid ? w4[w][s][j] : 0.f, acc[w][j][i], 0, 0, 0);
    }
  }

  auto finish = [&](int m, const Columns &g, const Columns &u) {
    if (m >= rows) return;
    const size_t at = (size_t)(m0 + m) * a.F + c;
    Columns h;
#pragma unroll
    for (int j = 0; j < C; ++j) h[j] = act_of<ACT>(g[j]) * u[j];
    auto put = [&](float *out, const Columns &value) {
      if (!out) return;
      if (c + C <= a.F) {
        *reinterpret_cast<ColumnsU *>(out + at) = value;
      } else {
#pragma unroll
        for (int j = 0; j < C - 1; ++j)
          if (c + j < a.F) out[at + j] = value[j];
      }
    };
    put(a.g, g);
    put(a.u, u);
    put(a.h, h);
  };
  auto first_row = [](int v) { return 32 * (v / 16) + 8 * (v % 16 / 4) + v % 4; };
  if (a.alone) {
#pragma unroll
    for (int v = 0; v < 16 * BLOCKS; ++v) {
      if (first_row(v) >= rows) continue;
      Columns of[2];
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int j = 0; j < C; ++j) of[w][j] = acc[w][j][v / 16][v % 16];
      finish(first_row(v) + 4 * half, of[0], of[1]);
    }
    return;
  }
  Columns sum[2][OWN];
#pragma unroll
  for (int round = 0; round < kWaves / ROUND; ++round) {
    if (first_row(round * ROUND * OWN) >= rows) break;  // uniform, as all that depends on rows below
    if (round) __syncthreads();
#pragma unroll
    for (int q = round * ROUND; q < (round + 1) * ROUND; ++q)
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        if (first_row(q * OWN + i) >= rows) continue;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          Columns o;
#pragma unroll
          for (int j = 0; j < C; ++j) o[j] = acc[w][j][(q * OWN + i) / 16][(q * OWN + i) % 16];
          if (wave == q) sum[w][i] = o;
          else part[q % ROUND][wave - (wave > q)][i][w][lane] = o;
        }
      }
    __syncthreads();
    if (wave / ROUND == round)
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        if (first_row(wave * OWN + i) >= rows) continue;
#pragma unroll
        for (int o = 0; o < kWaves - 1; ++o)
#pragma unroll
          for (int w = 0; w < 2; ++w) sum[w][i] += part[wave % ROUND][o][i][w][lane];
      }
  }
  if (a.pieces > 1) {
    constexpr int SC1 = 16;
    constexpr uint32_t kPieceBytes = 2u * kRows * kCols * 4u;
    const __amdgpu_buffer_rsrc_t pieces =
        make_rsrc(a.scratch + (size_t)group * a.pieces * (kPieceBytes / 4), (uint32_t)a.pieces * kPieceBytes);
    auto offset = [&](int p, int w, int i) {
      return (int)((uint32_t)p * kPieceBytes + (uint32_t)(((wave * OWN + i) * 2 + w) * 64 + lane) * (4u * C));
    };
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (first_row(wave * OWN + i) >= rows) continue;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        store_columns<SC1>(pieces, (uint32_t)offset(piece, w, i), sum[w][i]);
      }
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(a.tickets + group, 1u) == (unsigned)(a.pieces - 1);
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) a.tickets[group] = 0u;
#pragma unroll
    for (int i = 0; i < OWN; ++i) sum[0][i] = sum[1][i] = Columns{};
    // accumulators without a row were not written, and are not used
#pragma unroll 4
    for (int p = 0; p < a.pieces; ++p)
#pragma unroll
      for (int i = 0; i < OWN; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          sum[w][i] += load_columns<C, SC1>(pieces, first_row(wave * OWN + i) < rows ? (uint32_t)offset(p, w, i) : OOB);
        }
  }
#pragma unroll
  for (int i = 0; i < OWN; ++i) finish(first_row(wave * OWN + i) + 4 * half, sum[0][i], sum[1][i]);
}

// Up to four rows: vector multiply-adds.  Sixteen waves share 32 columns, eight lanes a row of the weights with four columns each, so
// that 4 096 columns already keep half of the CUs' loads going without a run of the reduction to be added across
// workgroups, which costs as long as reading 20 MB.  A longer reduction is better cut, from where on depends on where the weights
// come from.  This / cut, us, weights out of the last-level cache (the same ones again) and out of memory (700 MB of them in turn): one row of
// 1 024 x 4 096 5.7 / 10.6 and 11.0 / 12.3, 2 560 x 512 8.1 / 14.6 and 21.5 / 15.2, 4 096 x 512 10.2 / 19.4 and 32.8 / 20.1, 4 096 x 4 096
// 25.7 / 24.3 and 36.7 / 30.4; four rows of 1 000 x 2 731 9.2 / 11.1 and 13.7 / 12.2, 2 560 x 512 10.1 / 15.5 and 25.1 / 15.9.  The limit, one
// for one to four rows, is that of the cache, and part of the interface: up to it a call takes no scratch and can be captured.
constexpr int kFewest = 4, kNarrow = 32, kWide = 1024;
template <int ACT, int ROWS>
__global__ __launch_bounds__(kWide) void fewest_kernel(const Args a) {
  constexpr int WAVES = kWide / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = (by_neighbours(a.F) ? xcd_contiguous(blockIdx.x, gridDim.x) : (int)blockIdx.x) * kNarrow;
  const int c = c0 + 4 * (lane & 7);
  __shared__ f32x4v part[WAVES][2][ROWS][8];
  const uint32_t bytes = (uint32_t)a.K * (uint32_t)a.F * 4u;
  const __amdgpu_buffer_rsrc_t rsrc[2] = {make_rsrc(a.gate, bytes), make_rsrc(a.up, bytes)};
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, (uint32_t)a.M * (uint32_t)a.K * 4u);
  f32x4v acc[2][ROWS];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int m = 0; m < ROWS; ++m) acc[w][m] = f32x4v{0.f, 0.f, 0.f, 0.f};
  constexpr int DEPTH = ROWS > 2 ? 4 : 8;
  for (int k0 = wave * 8 + (lane >> 3); k0 < a.K; k0 += DEPTH * 8 * WAVES) {
    f32x4v wv[DEPTH][2];
    float xv[DEPTH][ROWS];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = k0 + d * 8 * WAVES;
      // columns past the end hold the next row's values, which are not stored
      const uint32_t off = k < a.K && c < a.F ? ((uint32_t)k * (uint32_t)a.F + (uint32_t)c) * 4u : OOB;
#pragma unroll
      for (int w = 0; w < 2; ++w) wv[d][w] = buf_load4(rsrc[w], off);
#pragma unroll
      for (int m = 0; m < ROWS; ++m) xv[d][m] = buf_load(xr, k < a.K ? ((uint32_t)m * (uint32_t)a.K + (uint32_t)k) * 4u : OOB);
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int m = 0; m < ROWS; ++m) acc[w][m] += xv[d][m] * wv[d][w];
  }
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[w][m][j] = lanes::sum<8>(acc[w][m][j]);
      if (lane < 8) part[wave][w][m][lane] = acc[w][m];
    }
  __syncthreads();
  const int m = threadIdx.x / kNarrow, n = c0 + (int)threadIdx.x % kNarrow;
  if (m >= ROWS || m >= a.M || n >= a.F) return;
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int o = 0; o < WAVES; ++o)
#pragma unroll
    for (int w = 0; w < 2; ++w) sum[w] += part[o][w][m][threadIdx.x % kNarrow / 4][threadIdx.x % 4];
  const size_t at = (size_t)m * a.F + n;
  if (a.g) {
    a.g[at] = sum[0];
    a.u[at] = sum[1];
  }
  if (a.h) a.h[at] = act_of<ACT>(sum[0]) * sum[1];
}

int64_t forward(int M, int K, int F, const float *x, const float *gate, const float *up, float *pre, float *h, int activation,
                hipStream_t s) {
  Args a{x, gate, up, pre, pre ? pre + (size_t)M * F : nullptr, h, M, K, F, cdiv(F, kCols), 0, 1, false, on_fp32(), on_fp32() ? K : 0, nullptr, nullptr};
  if (M <= kFewest && K <= 2560) {
    with_activation(activation, [&](auto act) {
      hipLaunchKernelGGL((M > 2 ? fewest_kernel<decltype(act)::value, 4> : M > 1 ? fewest_kernel<decltype(act)::value, 2> : fewest_kernel<decltype(act)::value, 1>),
                         dim3((unsigned)cdiv(F, kNarrow)), dim3(kWide), 0, s, a);
    });
    return 0;
  }
  const int rows = rows_of(M, F);
  // A strip a wave where the reduction is short and workgroups abound.  So / a strip a workgroup, us: 512 rows of 34 x 2 382 (304
  // workgroups) 17 / 27, 927 rows (570) 18 / 40; of 96 x 2 000, 512 rows (256) 20 / 16, 927 (480) 21 / 29; 512 of 200 x 4 000 (504) 31 / 36; 927
  // of 128 x 1 024 (240) 22 / 16.
  a.alone = K <= 256 && (int64_t)a.strips * cdiv(M, rows) > num_cus();
  const int64_t groups = (int64_t)(a.alone ? cdiv(a.strips, kWaves) : a.strips) * cdiv(M, rows);
  // about a workgroup a CU, a wave's run 32 reduction elements at least
  int pieces = (int)std::max<int64_t>(1, std::min<int64_t>({num_cus() / groups, K / (kWaves * 32), 32}));
  a.k_per_group = cdiv(K, pieces * kWaves * kGroup) * kWaves * kGroup;
  a.pieces = K ? cdiv(K, a.k_per_group) : 1;
  if (a.alone) {
    a.pieces = 1;
    a.k_per_group = std::max(K, 1);
  }
  if (a.pieces > 1) {
    const size_t bytes = (size_t)groups * a.pieces * 2 * rows * kCols * 4;
    if (being_captured(s)) return kCaptured;
    a.tickets = fold_tickets(s);
    a.scratch = a.tickets ? (float *)device_alloc(bytes, s) : nullptr;
    if (!a.scratch) return (int64_t)block_bytes(bytes);
  }
  with_activation(activation, [&](auto act) {
    hipLaunchKernelGGL((rows > 32 ? forward_kernel<decltype(act)::value, 2> : forward_kernel<decltype(act)::value, 1>),
                       dim3((unsigned)groups, (unsigned)a.pieces), dim3(kThreads), 0, s, a);
  });
  if (a.scratch) device_free(a.scratch, s);
  return 0;
}
// ---- the backward pass of little work, in one launch with nothing stored split ------------------------------------------
// Workgroups of dx (32 rows x 64 columns, along the inner axis, dg by gate and du by up in turn) and, behind them, of both weights'
// gradients (64 rows x 32 columns of each, along the rows).  dg and du are computed from g, u and dh wherever they are an operand.  Everything
// else is as in forward_kernel: a wave has a run of the reduction, its operands come from memory to registers and are split there, waves are
// added through LDS and workgroups by the last one.
struct BackwardArgs {
  const float *x, *gate, *up, *g, *u, *dh;  // no dh: g and u are dg and du
  float *dx, *dgate, *dup;                  // NULL: not wanted
  int M, K, F;
  struct Part {
    int tiles, cols, pieces, run;  // tiles in all and side by side; reduction elements of a workgroup, a multiple of kWaves * kGroup
    float *scratch;                // [tile][piece][accumulator of a lane][wave][lane]
    unsigned *tickets;
  } to_x, to_w;
  bool alone;  // every wave has a tile of the weights' gradients for itself, a workgroup four side by side
  bool exact;   // as above,
  int skipped;  // past any run's end
};

template <int ACT>
__device__ inline void projections_gradients(float g, float u, float d, float &dg, float &du) {
  if constexpr (ACT == kGiven) {
    dg = g;
    du = u;
  } else {
    Source::gradients<ACT>(g, u, d, dg, du);
  }
}

// Operands of a tile of dx: a, rows of dg and du, 32 of them; b, rows of the weights, 64 of them.
template <int ACT>
struct AlongInner {
  static constexpr int SUBS = 2, BLOCKS = 1;
  template <int COUNT>
  struct Raw {
    f32x4v d[3][COUNT / 4], w[2][2][COUNT / 4];
  };
  __amdgpu_buffer_rsrc_t d_rsrc[3], w_rsrc[2];
  uint32_t d_off, w_off[2];
  int half, k_end;
  __device__ inline AlongInner(const BackwardArgs &a, int m0, int c0, int k_end_, int lane) : half(lane >> 5), k_end(k_end_) {
    const uint32_t d_bytes = (uint32_t)a.M * (uint32_t)a.F * 4u, w_bytes = (uint32_t)a.K * (uint32_t)a.F * 4u;
    d_rsrc[0] = make_rsrc(a.g, d_bytes);
    d_rsrc[1] = make_rsrc(a.u, d_bytes);
    d_rsrc[2] = make_rsrc(ACT == kGiven ? nullptr : a.dh, ACT == kGiven ? 0u : d_bytes);
    w_rsrc[0] = make_rsrc(a.gate, w_bytes);
    w_rsrc[1] = make_rsrc(a.up, w_bytes);
    const int m = m0 + (lane & 31);
    d_off = m < a.M ? (uint32_t)m * (uint32_t)a.F * 4u : OOB;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = c0 + 32 * j + (lane & 31);
      w_off[j] = k < a.K ? (uint32_t)k * (uint32_t)a.F * 4u : OOB;
    }
  }
  template <int COUNT>
  __device__ inline void load(int k0, Raw<COUNT> &raw) const {
    // behind the run's end what is there already, which counts as zero
    const int from = (k0 < k_end ? k0 : max(k_end - 2 * COUNT, 0)) * 4;
    auto four = [&](__amdgpu_buffer_rsrc_t r, uint32_t off) {
      return __builtin_bit_cast(f32x4v, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, from, 0));
    };
#pragma unroll
    for (int s = 0; s < COUNT / 4; ++s) {
      const uint32_t at = (uint32_t)(COUNT * half + 4 * s) * 4u;
#pragma unroll
      for (int w = 0; w < (ACT == kGiven ? 2 : 3); ++w) raw.d[w][s] = four(d_rsrc[w], d_off + at);
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int j = 0; j < 2; ++j) raw.w[w][j][s] = four(w_rsrc[w], w_off[j] + at);
    }
  }
  // EXACT: what counts as zero is zero in both, for the weights may hold an infinity there
  template <bool EXACT, int COUNT>
  __device__ inline void operands(int k0, const Raw<COUNT> &raw, float (&a)[SUBS][BLOCKS][COUNT], float (&b)[SUBS][2][COUNT]) const {
    const int valid = k_end - k0 - COUNT * half;
#pragma unroll
    for (int s = 0; s < COUNT; ++s) {
      float dg, du;
      projections_gradients<ACT>(raw.d[0][s / 4][s % 4], raw.d[1][s / 4][s % 4], ACT == kGiven ? 0.f : raw.d[2][s / 4][s % 4], dg, du);
      a[0][0][s] = s < valid ? dg : 0.f;
      a[1][0][s] = s < valid ? du : 0.f;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int j = 0; j < 2; ++j) b[w][j][s] = !EXACT || s < valid ? raw.w[w][j][s / 4][s % 4] : 0.f;
    }
  }
};

// Operands of a tile of the weights' gradients: a, 64 columns of x, two neighbours a lane; b, 32 columns of dg and of du.
template <int ACT>
struct AlongRows {
  static constexpr int SUBS = 1, BLOCKS = 2;
  template <int COUNT>
  struct Raw {
    split::f32x2v x[COUNT];
    float d[3][COUNT];
  };
  __amdgpu_buffer_rsrc_t x_rsrc, d_rsrc[3];
  uint32_t x_off, d_off, x_row, d_row;
  int half, k_end;
  __device__ inline AlongRows(const BackwardArgs &a, int k0, int f0, int k_end_, int lane) : half(lane >> 5), k_end(k_end_) {
    x_row = (uint32_t)a.K * 4u;
    d_row = (uint32_t)a.F * 4u;
    x_rsrc = make_rsrc(a.x, (uint32_t)k_end * x_row);  // behind the run's end: zeros
    d_rsrc[0] = make_rsrc(a.g, (uint32_t)k_end * d_row);
    d_rsrc[1] = make_rsrc(a.u, (uint32_t)k_end * d_row);
    d_rsrc[2] = make_rsrc(ACT == kGiven ? nullptr : a.dh, ACT == kGiven ? 0u : (uint32_t)k_end * d_row);
    const int k = k0 + 2 * (lane & 31), f = f0 + (lane & 31);
    x_off = k < a.K ? (uint32_t)k * 4u : OOB;
    d_off = f < a.F ? (uint32_t)f * 4u : OOB;
  }
  template <int COUNT>
  __device__ inline void load(int k0, Raw<COUNT> &raw) const {
#pragma unroll
    for (int s = 0; s < COUNT; ++s) {
      const uint32_t row = (uint32_t)min(k0 + COUNT * half + s, k_end);
      raw.x[s] = __builtin_bit_cast(split::f32x2v, __builtin_amdgcn_raw_buffer_load_b64(x_rsrc, (int)(x_off + row * x_row), 0, 0));
#pragma unroll
      for (int w = 0; w < (ACT == kGiven ? 2 : 3); ++w) raw.d[w][s] = buf_load(d_rsrc[w], d_off + row * d_row);
    }
  }
  template <bool EXACT, int COUNT>
  __device__ inline void operands(int, const Raw<COUNT> &raw, float (&a)[SUBS][BLOCKS][COUNT], float (&b)[SUBS][2][COUNT]) const {
#pragma unroll
    for (int s = 0; s < COUNT; ++s) {
      a[0][0][s] = raw.x[s][0];
      a[0][1][s] = raw.x[s][1];
      projections_gradients<ACT>(raw.d[0][s], raw.d[1][s], ACT == kGiven ? 0.f : raw.d[2][s], b[0][0][s], b[0][1][s]);
    }
  }
};

// A tile's sums over one wave's run.
template <class From>
__device__ __forceinline__ void run_of_wave(const From &from, const BackwardArgs &args, int k_begin, int k_end, f32x16 (&acc)[From::BLOCKS][2]) {
  constexpr int BLOCKS = From::BLOCKS, SUBS = From::SUBS;
  f32x16 low[BLOCKS][2];
  auto clear = [](f32x16 (&sums)[BLOCKS][2]) {
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[i][j][v] = 0.f;
  };
  clear(acc);
  clear(low);
  typename From::template Raw<8> raw[kDepth];
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    from.load(k_begin + kGroup * d, raw[d]);
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int k0 = k_begin + args.skipped; k0 < k_end; k0 += kGroup * kDepth)
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      float a[SUBS][BLOCKS][8], b[SUBS][2][8];
      from.template operands<false>(k0 + kGroup * d, raw[d], a, b);
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub) {
        split::bf16x8 as[BLOCKS][3];
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i) {
          const Slices slices([&](int k) { return a[sub][i][k]; });
#pragma unroll
          for (int q = 0; q < 3; ++q) as[i][q] = slices.of[q];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const Slices bs([&](int k) { return b[sub][j][k]; });
#pragma unroll
          for (int p = 0; p < 6; ++p) {
            constexpr int of_a[6] = {0, 0, 1, 0, 1, 2}, of_b[6] = {0, 1, 0, 2, 1, 0};
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) {
              f32x16 &sum = p == 0 ? acc[i][j] : low[i][j];
              sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as[i][of_a[p]], bs.of[of_b[p]], sum, 0, 0, 0);
            }
          }
        }
      }
      from.load(k0 + kGroup * (d + kDepth), raw[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  float finite = 0.f;
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        acc[i][j][v] = (acc[i][j][v] + low[i][j][v]) * split::kUnscale;
        finite = __builtin_fmaf(acc[i][j][v], 0.f, finite);
      }
  if (!args.exact && !__any(finite != finite)) return;
  clear(acc);
#pragma unroll 1
  for (int k0 = k_begin; k0 < k_end; k0 += 8) {
    typename From::template Raw<4> few_raw;
    float a[SUBS][BLOCKS][4], b[SUBS][2][4];
    from.load(k0, few_raw);
    from.template operands<true>(k0, few_raw, a, b);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
        for (int i = 0; i < BLOCKS; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[sub][i][s], b[sub][j][s], acc[i][j], 0, 0, 0);
  }
}

// The waves' sums added, and the pieces'; wave q then holds accumulators 4 q .. 4 q + 3 of every block, rows 8 q + 4 half + e.  False in
// workgroups that have nothing left to do.
template <int N>
__device__ __forceinline__ bool join(const f32x16 (&acc)[N / 2][2], float *part, unsigned &last, const BackwardArgs::Part &p, int tile,
                                     int piece, int wave, int lane, float (&own)[N][4]) {
#pragma unroll
  for (int q = 0; q < kWaves; ++q)
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = acc[b / 2][b % 2][4 * q + e];
        if (wave == q) own[b][e] = v;
        else part[((q * (kWaves - 1) + wave - (wave > q)) * 4 * N + b * 4 + e) * 64 + lane] = v;
      }
  __syncthreads();
#pragma unroll
  for (int o = 0; o < kWaves - 1; ++o)
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) own[b][e] += part[((wave * (kWaves - 1) + o) * 4 * N + b * 4 + e) * 64 + lane];
  if (p.pieces == 1) return true;
  constexpr int SC1 = 16;
  constexpr uint32_t kPieceBytes = 4u * N * kThreads * 4u;
  const __amdgpu_buffer_rsrc_t pieces = make_rsrc(p.scratch + (size_t)tile * p.pieces * (kPieceBytes / 4), (uint32_t)p.pieces * kPieceBytes);
  auto offset = [&](int of, int b) { return (uint32_t)of * kPieceBytes + (uint32_t)((b * kWaves + wave) * 64 + lane) * 16u; };
#pragma unroll
  for (int b = 0; b < N; ++b) {
    const f32x4v v = {own[b][0], own[b][1], own[b][2], own[b][3]};
    store_columns<SC1>(pieces, offset(piece, b), v);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.tickets + tile, 1u) == (unsigned)(p.pieces - 1);
  __syncthreads();
  if (!last) return false;
  if (threadIdx.x == 0) p.tickets[tile] = 0u;
  f32x4v sum[N] = {};
#pragma unroll 4
  for (int of = 0; of < p.pieces; ++of)
#pragma unroll
    for (int b = 0; b < N; ++b) sum[b] += load_columns<4, SC1>(pieces, offset(of, b));
#pragma unroll
  for (int b = 0; b < N; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) own[b][e] = sum[b][e];
  return true;
}

template <int ACT>
__global__ __launch_bounds__(kThreads, 2) void backward_kernel(const BackwardArgs a) {
  __shared__ float part[kWaves * (kWaves - 1) * 4 * 4 * 64];
  __shared__ unsigned last;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, along = lane & 31;
  const int x_groups = a.to_x.tiles * a.to_x.pieces;
  if ((int)blockIdx.x < x_groups) {
    const int tile = blockIdx.x % a.to_x.tiles, piece = blockIdx.x / a.to_x.tiles;
    const int m0 = tile / a.to_x.cols * 32, c0 = tile % a.to_x.cols * 64;
    const int k_begin = piece * a.to_x.run + wave * (a.to_x.run / kWaves), k_end = min(a.F, k_begin + a.to_x.run / kWaves);
    f32x16 acc[1][2];
    run_of_wave(AlongInner<ACT>(a, m0, c0, k_end, lane), a, k_begin, k_end, acc);
    float own[2][4];
    if (!join<2>(acc, part, last, a.to_x, tile, piece, wave, lane, own)) return;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + 8 * wave + 4 * half + e, k = c0 + 32 * b + along;
        if (m < a.M && k < a.K) a.dx[(size_t)m * a.K + k] = own[b][e];
      }
    return;
  }
  const int group = (int)blockIdx.x - x_groups;
  const int tile = a.alone ? group * kWaves + wave : group % a.to_w.tiles, piece = a.alone ? 0 : group / a.to_w.tiles;
  const int c0 = tile / a.to_w.cols * 64, f0 = tile % a.to_w.cols * 32;
  const int of_wave = a.alone ? a.to_w.run : a.to_w.run / kWaves;
  const int k_begin = a.alone ? 0 : piece * a.to_w.run + wave * of_wave, k_end = min(a.M, k_begin + of_wave);
  f32x16 acc[2][2];
  run_of_wave(AlongRows<ACT>(a, c0, f0, k_end, lane), a, k_begin, k_end, acc);
  auto put = [&](int b, int row, float v) {
    float *out = b % 2 ? a.dup : a.dgate;
    const int k = c0 + 2 * row + b / 2, f = f0 + along;
    if (out && k < a.K && f < a.F) out[(size_t)k * a.F + f] = v;
  };
  if (a.alone) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int v = 0; v < 16; ++v) put(b, 8 * (v / 4) + 4 * half + v % 4, acc[b / 2][b % 2][v]);
    return;
  }
  float own[4][4];
  if (!join<4>(acc, part, last, a.to_w, tile, piece, wave, lane, own)) return;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) put(b, 8 * wave + 4 * half + e, own[b][e]);
}

int64_t backward(int M, int K, int F, const float *x, const float *gate, const float *up, const Source &d, float *dx, float *dgate,
                 float *dup, hipStream_t s) {
  BackwardArgs a{x, gate, up, d.p[0], d.p[1], d.dh, dx, dgate, dup, M, K, F, {}, {}, false, on_fp32(), on_fp32() ? 1 << 29 : 0};
  // pieces as for all three gradients, so that each has the same bits alone
  auto part = [](int rows, int cols, int steps) {
    BackwardArgs::Part p{rows * cols, cols, 1, 0, nullptr, nullptr};
    const int pieces = std::max(1, std::min({num_cus() / std::max(p.tiles, 1), steps / (kWaves * 2 * kGroup), 32}));
    p.run = std::max(1, cdiv(steps, pieces * kWaves * kGroup)) * kWaves * kGroup;
    p.pieces = std::max(1, cdiv(steps, p.run));
    return p;
  };
  a.to_x = part(cdiv(M, 32), cdiv(K, 64), F);
  a.to_w = part(cdiv(K, 64), cdiv(F, 32), M);
  // A tile a wave where four waves would have a group each at most, or workgroups abound.  So / a tile a workgroup, us: 64 rows of
  // 512 x 1 376 (344 tiles) 16.8 / 19.1, 128 rows 24.4 / 22.8; 128 rows of 1 000 x 1 537 (784) 37 / 40; 24 rows of 1 024 x 4 096 (2 048) 28 / 49.
  a.alone = M <= kWaves * kGroup || a.to_w.tiles >= 2 * num_cus();
  if (a.alone) {
    a.to_w.run = M;
    a.to_w.pieces = 1;
  }
  if (!dx) a.to_x.tiles = 0;
  if (!dgate && !dup) a.to_w.tiles = 0;
  Layout l;
  const size_t x_at = a.to_x.pieces > 1 ? l.take((size_t)a.to_x.tiles * a.to_x.pieces * 32 * 64 * 4) : 0;
  const size_t w_at = a.to_w.pieces > 1 ? l.take((size_t)a.to_w.tiles * a.to_w.pieces * 64 * 64 * 4) : 0;
  char *base = nullptr;
  if (l.bytes) {
    unsigned *tickets = fold_tickets(s);
    base = tickets ? (char *)device_alloc(l.bytes, s) : nullptr;
    if (!base) return (int64_t)block_bytes(l.bytes);
    a.to_x.scratch = (float *)(base + x_at);
    a.to_w.scratch = (float *)(base + w_at);
    a.to_x.tickets = tickets;
    a.to_w.tickets = tickets + kFoldTicketSlots / 2;
  }
  const unsigned groups = (unsigned)(a.to_x.tiles * a.to_x.pieces + (a.alone ? cdiv(a.to_w.tiles, kWaves) : a.to_w.tiles * a.to_w.pieces));
  if (groups == 0) return 0;
  auto go = [&](auto act) {
    hipLaunchKernelGGL(backward_kernel<decltype(act)::value>, dim3(groups), dim3(kThreads), 0, s, a);
  };
  if (d.dh) with_activation(d.activation, go);
  else go(std::integral_constant<int, kGiven>{});
  if (base) device_free(base, s);
  return 0;
}
}  // namespace few

unsigned vectors_grid(int64_t count) { return (unsigned)((count + 4 * kThreads - 1) / (4 * kThreads)); }

bool is_pair(const DLArray *pre, const DLArray *one) {
  return pre->ndim == one->ndim + 1 && pre->shape[0] == 2 &&
         std::equal(one->shape, one->shape + one->ndim, pre->shape + 1);
}

int geometry(const char *what, const DLArray *x, const DLArray *gate, const DLArray *up, int activation, int64_t &M,
             int64_t &K, int64_t &F) {
  auto fail = [&](const char *why) {
    fprintf(stderr, "[tinyflow_amd] %s: %s\n", what, why);
    return -1;
  };
  if (!on_gpu(x) || !on_gpu(gate) || !on_gpu(up)) return fail("arrays must live on the GPU");
  if (x->ndim != 2 || gate->ndim != 2 || !same_shape(gate, up)) return fail("input and the two weights of one shape must be 2-D");
  M = x->shape[0];
  K = x->shape[1];
  F = gate->shape[1];
  if (gate->shape[0] != K) return fail("the weights must have a row for each of the input's columns");
  if (activation < kSigmoid || activation > kGelu) return fail("unknown activation");
  const int64_t most = ((int64_t)1 << 29) - 1;
  if (M > most || K > most || F > most || M * K > most || K * F > most || M * F > most)
    return fail("arrays of 2 GiB or more are not supported");
  if (M > 1 << 26 || F > 1 << 26) return fail("more than 2^26 rows or columns are not supported");
  return 0;
}

}  // namespace

extern "C" int DLGpuGatedActivation(const DLArrayHandle pre, DLArrayHandle output, int activation, void **stream) {
  TF_REQUIRE(on_gpu(pre) && on_gpu(output), "arrays must live on the GPU");
  TF_REQUIRE(is_pair(pre, output), "pre must hold two arrays of the output's shape");
  TF_REQUIRE(activation >= kSigmoid && activation <= kGelu, "unknown activation %d", activation);
  TF_REQUIRE(same_device({pre, output}), "arrays must live on one device");
  TF_REQUIRE(!overlaps(pre, output), "output must not overlap pre");
  const int64_t n = numel(output);
  TF_REQUIRE(n < (int64_t)1 << 33, "2^33 elements or more are not supported");
  announce_write(output);
  hipStream_t s = stream_of(stream);
  if (n == 0) return 0;
  const float *g = (const float *)pre->data;
  with_activation(activation, [&](auto act) {
    hipLaunchKernelGGL(activation_kernel<decltype(act)::value>, dim3(vectors_grid(n)), dim3(kThreads), 0, s, g, g + n,
                       (float *)output->data, n);
  });
  return finish(s, "DLGpuGatedActivation");
}

extern "C" int DLGpuGatedActivationBackward(const DLArrayHandle pre, const DLArrayHandle doutput, DLArrayHandle dpre,
                                            int activation, void **stream) {
  TF_REQUIRE(on_gpu(pre) && on_gpu(doutput) && on_gpu(dpre), "arrays must live on the GPU");
  TF_REQUIRE(is_pair(pre, doutput) && same_shape(pre, dpre), "pre and dpre must hold two arrays of doutput's shape");
  TF_REQUIRE(activation >= kSigmoid && activation <= kGelu, "unknown activation %d", activation);
  TF_REQUIRE(same_device({pre, doutput, dpre}), "arrays must live on one device");
  TF_REQUIRE(!overlaps(dpre, doutput) && (pre->data == dpre->data || !overlaps(pre, dpre)),
             "dpre must be pre or overlap neither pre nor doutput");
  const int64_t n = numel(doutput);
  TF_REQUIRE(n < (int64_t)1 << 33, "2^33 elements or more are not supported");
  announce_write(dpre);
  hipStream_t s = stream_of(stream);
  if (n == 0) return 0;
  const float *g = (const float *)pre->data;
  float *d = (float *)dpre->data;
  with_activation(activation, [&](auto act) {
    hipLaunchKernelGGL(activation_backward_kernel<decltype(act)::value>, dim3(vectors_grid(n)), dim3(kThreads), 0, s, g, g + n,
                       (const float *)doutput->data, d, d + n, n);
  });
  return finish(s, "DLGpuGatedActivationBackward");
}

extern "C" int DLGpuGatedFeedForward(const DLArrayHandle input, const DLArrayHandle gate, const DLArrayHandle up,
                                     DLArrayHandle pre, DLArrayHandle output, int activation, int *memorytoSaving,
                                     void **stream) {
  int64_t M, K, F;
  if (geometry(__func__, input, gate, up, activation, M, K, F) != 0) return -1;
  TF_REQUIRE(pre || output, "no result is asked for");
  TF_REQUIRE(!output || (on_gpu(output) && output->ndim == 2 && output->shape[0] == M && output->shape[1] == F),
             "output must live on the GPU and be %lld x %lld", (long long)M, (long long)F);
  TF_REQUIRE(!pre || (on_gpu(pre) && pre->ndim == 3 && pre->shape[0] == 2 && pre->shape[1] == M && pre->shape[2] == F),
             "pre must live on the GPU and be 2 x %lld x %lld", (long long)M, (long long)F);
  TF_REQUIRE(same_device({input, gate, up, pre, output}), "arrays must live on one device");
  for (const DLArray *written : {(const DLArray *)pre, (const DLArray *)output})
    for (const DLArray *read : {(const DLArray *)input, (const DLArray *)gate, (const DLArray *)up})
      TF_REQUIRE(!overlaps(read, written), "results must not overlap what they are computed from");
  TF_REQUIRE(!overlaps(pre, output), "results must not overlap");
  if (pre) announce_write(pre);
  if (output) announce_write(output);
  hipStream_t s = stream_of(stream);
  if (M == 0 || F == 0) return 0;
  const int64_t wanted = (forward_on_pairs(M, K, F) ? forward_by_pairs : few::forward)(
      (int)M, (int)K, (int)F, (const float *)input->data, (const float *)gate->data, (const float *)up->data,
      pre ? (float *)pre->data : nullptr, output ? (float *)output->data : nullptr, activation, s);
  TF_REQUIRE(wanted != kCaptured, "the call takes scratch, which a captured stream cannot give back");
  if (wanted && memorytoSaving) *memorytoSaving = shortfall((size_t)wanted);
  return wanted ? 0 : finish(s, "DLGpuGatedFeedForward");
}

extern "C" int DLGpuGatedFeedForwardBackward(const DLArrayHandle input, const DLArrayHandle gate, const DLArrayHandle up,
                                             const DLArrayHandle pre, const DLArrayHandle doutput, DLArrayHandle dinput,
                                             DLArrayHandle dgate, DLArrayHandle dup, int activation, int *memorytoSaving,
                                             void **stream) {
  int64_t M, K, F;
  if (geometry(__func__, input, gate, up, activation, M, K, F) != 0) return -1;
  auto is_stacked = [&](const DLArray *a) {
    return on_gpu(a) && a->ndim == 3 && a->shape[0] == 2 && a->shape[1] == M && a->shape[2] == F;
  };
  TF_REQUIRE(!pre || is_stacked(pre), "pre must live on the GPU and be 2 x %lld x %lld", (long long)M, (long long)F);
  if (pre)
    TF_REQUIRE(on_gpu(doutput) && doutput->ndim == 2 && doutput->shape[0] == M && doutput->shape[1] == F,
               "doutput must live on the GPU and be %lld x %lld", (long long)M, (long long)F);
  else
    TF_REQUIRE(is_stacked(doutput), "doutput without pre must live on the GPU and be 2 x %lld x %lld", (long long)M, (long long)F);
  TF_REQUIRE(dinput || dgate || dup, "no gradient is asked for");
  TF_REQUIRE(!dinput || (on_gpu(dinput) && same_shape(dinput, input)), "dinput must live on the GPU and have the input's shape");
  TF_REQUIRE(!dgate || (on_gpu(dgate) && same_shape(dgate, gate)), "dgate must live on the GPU and have the weights' shape");
  TF_REQUIRE(!dup || (on_gpu(dup) && same_shape(dup, gate)), "dup must live on the GPU and have the weights' shape");
  TF_REQUIRE(same_device({input, gate, up, pre, doutput, dinput, dgate, dup}), "arrays must live on one device");
  for (const DLArray *written : {(const DLArray *)dinput, (const DLArray *)dgate, (const DLArray *)dup})
    for (const DLArray *read : {(const DLArray *)input, (const DLArray *)gate, (const DLArray *)up, (const DLArray *)pre,
                                (const DLArray *)doutput})
      TF_REQUIRE(!overlaps(read, written), "gradients must not overlap what they are computed from");
  TF_REQUIRE(!overlaps(dinput, dgate) && !overlaps(dinput, dup) && !overlaps(dgate, dup), "gradients must not overlap");
  for (const DLArray *written : {(const DLArray *)dinput, (const DLArray *)dgate, (const DLArray *)dup}) announce_write(written);
  hipStream_t s = stream_of(stream);
  TF_REQUIRE(!being_captured(s), "the call takes scratch, which a captured stream cannot give back");
  const float *g = pre ? (const float *)pre->data : (const float *)doutput->data;
  const Source d{{g, g + M * F}, pre ? (const float *)doutput->data : nullptr, (int)M, (int)F, pre ? activation : kGiven};
  const int64_t wanted = (backward_on_pairs(M, K, F) ? backward_by_pairs : few::backward)(
      (int)M, (int)K, (int)F, (const float *)input->data, (const float *)gate->data, (const float *)up->data, d,
      dinput ? (float *)dinput->data : nullptr, dgate ? (float *)dgate->data : nullptr, dup ? (float *)dup->data : nullptr, s);
  if (wanted && memorytoSaving) *memorytoSaving = shortfall((size_t)wanted);
  return wanted ? 0 : finish(s, "DLGpuGatedFeedForwardBackward");
}
