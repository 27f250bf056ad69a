// Layer norm over the last axis, forward and backward (no counterpart in the reference, whose only norm is the batch
// norm of bn.hip).
//
//   mu = mean(x), v = mean((x - mu)^2), s = 1 / sqrt(v + eps), xh = (x - mu) s
//   y  = gamma xh + beta
//   a  = gamma dy,  dx = s (a - mean(a) - xh mean(a xh)),  dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// Nothing is kept between the two passes: the backward pass has the row of x in registers anyway and computes mu and s
// again from there, which moves no byte, and neither pass depends on the other having run.
//
// Bound: HBM.  A row is read once into registers, by a wave or by as many waves as it takes, and both
// statistics are taken from there, the squares after the mean is known (a sum of x^2 would cancel where the mean is
// large).  The mean of fp32 sums is off by a few steps of its own last place, which next to a small spread is a large part of it (constant
// rows of up to 1 000 in 5 000 columns: y off by up to 0.16).  So the deviations d = x - m from that first mean m are summed along with their
// squares: with e = mean(d), mu = m + e and v = mean(d^2) - e^2, where next to nothing cancels, and xh = (d - e) s.  What is left is off by
// steps of the deviations' last place.  All sums are fp32; their order depends on the shape alone.
#include "internal.h"
#include "lanes.h"

#include <algorithm>
#include <type_traits>

using namespace tf;

namespace {

template <int V>
using IC = std::integral_constant<int, V>;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));  // rows of any length start anywhere: 16-byte accesses on 4-byte alignment

// Sum over the T lanes that share a row; `room` is T / 64 floats of that row's that nothing else uses until the next barrier but
// one.  Rows of several waves pass a barrier: all rows of a workgroup get here together.
template <int T>
__device__ inline float row_sum(float v, float *room) {
  v = lanes::sum(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) room[threadIdx.x % T / 64] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += room[w];
  }
  return v;
}

// Two sums at once.
template <int T>
__device__ inline void row_sums(float &a, float &b, float (*room)[2]) {
  a = lanes::sum(a);
  b = lanes::sum(b);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) {
      room[threadIdx.x % T / 64][0] = a;
      room[threadIdx.x % T / 64][1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
      a += room[w][0];
      b += room[w][1];
    }
  }
}

// VPT vectors of a row in the registers of T lanes: vector e of lane l holds columns 4 (e T + l) and the three behind it;
// columns past the row's end read as zero and are not written.
template <int T, int VPT>
struct Row {
  f32x4 v[VPT];
  __device__ inline void load(const float *__restrict__ row, int cols, int lane) {
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
      const int c = 4 * (e * T + lane);
      v[e] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (c + 4 <= cols) {
        v[e] = *reinterpret_cast<const f32x4u *>(row + c);
      } else if (c < cols) {
        v[e][0] = row[c];
        if (c + 1 < cols) v[e][1] = row[c + 1];
        if (c + 2 < cols) v[e][2] = row[c + 2];
      }
    }
  }
  template <bool PAST = false>
  __device__ inline void store(float *__restrict__ row, int cols, int lane) const {
#pragma unroll
    for (int e = 0; e < VPT; ++e) {
      const int c = 4 * (e * T + lane);
      if (c + 4 <= cols) {
        if (PAST) __builtin_nontemporal_store(v[e], reinterpret_cast<f32x4u *>(row + c));
        else *reinterpret_cast<f32x4u *>(row + c) = v[e];
      } else if (c < cols) {
        row[c] = v[e][0];
        if (c + 1 < cols) row[c + 1] = v[e][1];
        if (c + 2 < cols) row[c + 2] = v[e][2];
      }
    }
  }
  __device__ inline float sum() const {
    f32x4 s = v[0];
#pragma unroll
    for (int e = 1; e < VPT; ++e) s += v[e];
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
  // v - m inside the row, zero past its end
  __device__ inline void subtract(float m, int cols, int lane) {
#pragma unroll
    for (int e = 0; e < VPT; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[e][i] = 4 * (e * T + lane) + i < cols ? v[e][i] - m : 0.f;
  }
  __device__ inline float dot(const Row &o) const {
    f32x4 s = v[0] * o.v[0];
#pragma unroll
    for (int e = 1; e < VPT; ++e) s += v[e] * o.v[e];
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
};

// From the sums of a row's deviations d from its first mean and of their squares: xh = d s - es.
struct Spread {
  float s, es;
  __device__ inline Spread(float sum, float square_sum, float n, float eps) {
    const float e = sum / n, v = square_sum / n - e * e;
    s = 1.f / sqrtf((v < 0.f ? 0.f : v) + eps);  // a NaN stays one
    es = e * s;
  }
};

// Workgroups as a grid none of whose dimensions, times the workgroup, passes 2^32.
dim3 grid_of(int64_t groups) { return dim3((unsigned)std::min<int64_t>(groups, 1 << 20), (unsigned)((groups + (1 << 20) - 1) >> 20)); }
__device__ inline int64_t group_index() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// T lanes a row, WG / T rows a workgroup.  y may be x, here and below.
template <int T, int VPT, bool PAST>
__global__ __launch_bounds__(T > 256 ? T : 256) void forward_kernel(const float *x, const float *__restrict__ gamma,
                                                                  const float *__restrict__ beta, float *y,
                                                                  int64_t rows, int cols, float n, float eps) {
  constexpr int WG = T > 256 ? T : 256;
  __shared__ float room[T / 64], rooms[T / 64][2];
  const int lane = threadIdx.x % T;
  const int64_t r = group_index() * (WG / T) + threadIdx.x / T;
  if (r >= rows) return;  // whole waves, and no barrier where several rows share a workgroup
  Row<T, VPT> row, g, b;
  row.load(x + r * cols, cols, lane);
  g.load(gamma, cols, lane);
  b.load(beta, cols, lane);
  row.subtract(row_sum<T>(row.sum(), room) / n, cols, lane);
  float sum = row.sum(), squares = row.dot(row);
  row_sums<T>(sum, squares, rooms);
  const Spread of(sum, squares, n, eps);
#pragma unroll
  for (int e = 0; e < VPT; ++e) row.v[e] = (row.v[e] * of.s - of.es) * g.v[e] + b.v[e];
  row.template store<PAST>(y + r * cols, cols, lane);
}

// Rows that do not fit registers: three passes, the later two mostly out of the caches, of four bytes a lane and load.  What bounds them is
// a workgroup's latency, pass behind pass: 300 x 40 003 43 us (2.2 TB/s of what is needed), dx 63, all gradients 95; 1 000 x 17 000 42 and
// 101, where 1 000 x 16 000 in registers takes 64 backward.  No model has rows of that length; the forms are there for the interface's range.
constexpr int kLong = 1024;

// f(column, sums) over a lane's columns of a row, in runs of kRun with sums of their own: of 2^26 columns no sum has more than 512 members.
// One after the other the 65 536 of a lane leave the mean of a row of 777.7 at 777.25.
constexpr int kRun = 256;
template <class F>
__device__ inline void sum_columns(int cols, float (&sums)[2], F &&f) {
  sums[0] = sums[1] = 0.f;
  for (int c0 = threadIdx.x; c0 < cols; c0 += kRun * kLong) {
    float run[2] = {0.f, 0.f};
    const int end = min(cols, c0 + kRun * kLong);
    for (int c = c0; c < end; c += kLong) f(c, run);
    sums[0] += run[0];
    sums[1] += run[1];
  }
}

// A long row's first mean and its spread about it.
__device__ inline Spread long_spread(const float *row, int cols, float n, float eps, float (*rooms)[kLong / 64][2], float &mean) {
  float sums[2];
  sum_columns(cols, sums, [&](int c, float (&run)[2]) { run[0] += row[c]; });
  row_sums<kLong>(sums[0], sums[1], rooms[0]);
  const float m = mean = sums[0] / n;
  sum_columns(cols, sums, [&](int c, float (&run)[2]) {
    const float d = row[c] - m;
    run[0] += d;
    run[1] += d * d;
  });
  row_sums<kLong>(sums[0], sums[1], rooms[1]);
  return Spread(sums[0], sums[1], n, eps);
}

__global__ __launch_bounds__(kLong) void forward_long_kernel(const float *x, const float *__restrict__ gamma,
                                                            const float *__restrict__ beta, float *y,
                                                            int64_t rows, int cols, float n, float eps) {
  __shared__ float rooms[2][kLong / 64][2];
  if (group_index() >= rows) return;
  const float *row = x + group_index() * cols;
  float mean;
  const Spread of = long_spread(row, cols, n, eps, rooms, mean);
  float *out = y + group_index() * cols;
  for (int c = threadIdx.x; c < cols; c += kLong) out[c] = ((row[c] - mean) * of.s - of.es) * gamma[c] + beta[c];
}

// Columns of a partial sum in memory: whole lines of kSumCols, so that a workgroup that adds them reads no neighbour's: 5 003 x 1 537 23.8 ->
// 23.4 us.
constexpr int kSumCols = 32;
__host__ __device__ inline int64_t padded(int64_t cols) { return (cols + kSumCols - 1) / kSumCols * kSumCols; }

// Rows blockIdx.x * (WG / T) + ..., then gridDim.x * (WG / T) further on, and so on, the next one on its way while one is worked
// on where PARAMS: without, workgroups have a row of each of their WG / T, and the registers are too few for a second one in the longest rows
// (us with it / without: 1 000 x 16 000 45 / 37.6, 2 000 x 8 000 44 / 31.6, 4 096 x 1 024 7.2 / 6.3).  With PARAMS every lane
// keeps the sums of dy xh and dy of its columns over the rows that it sees.  At the end the workgroup's rows are added through LDS, in
// their order, and go to partial[blockIdx.x][2][padded(cols)].
template <int T, int VPT, int WG, bool PARAMS, bool PAST>
__global__ __launch_bounds__(WG) void backward_kernel(const float *__restrict__ x, const float *__restrict__ gamma,
                                                    const float *__restrict__ dy, float *__restrict__ dx,
                                                    float *__restrict__ partial, int64_t rows, int cols, float n, float eps) {
  constexpr int ROWS = WG / T;
  constexpr bool HOLD = T * VPT < 4096;  // gamma in registers; else from the caches, row by row
  __shared__ float rooms[ROWS][3][T / 64][2];
  const int lane = threadIdx.x % T, sub = threadIdx.x / T;
  auto &room = rooms[sub];
  const int64_t step = (int64_t)gridDim.x * ROWS;
  Row<T, VPT> g, dgamma, dbeta, xh, d;
  if (dx && HOLD) g.load(gamma, cols, lane);
#pragma unroll
  for (int e = 0; e < VPT; ++e) dgamma.v[e] = dbeta.v[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  // a row behind the last one is worked on for the barriers' sake, on the last one's values, and left out of everything
  auto load = [&](int64_t r, Row<T, VPT> &of_x, Row<T, VPT> &of_dy) {
    r = r < rows ? r : rows - 1;
    of_x.load(x + r * cols, cols, lane);
    of_dy.load(dy + r * cols, cols, lane);
  };
  int64_t first = (int64_t)blockIdx.x * ROWS;
  if (PARAMS && first < rows) load(first + sub, xh, d);
  for (; first < rows; first += step) {
    const int64_t r = first + sub;
    const bool live = r < rows;  // of whole waves
    Row<T, VPT> next_x, next_d;
    if (!PARAMS) load(r, xh, d);
    else if (first + step < rows) load(r + step, next_x, next_d);
    xh.subtract(row_sum<T>(xh.sum(), &room[0][0][0]) / n, cols, lane);
    float sum = xh.sum(), squares = xh.dot(xh);
    row_sums<T>(sum, squares, room[1]);
    const Spread of(sum, squares, n, eps);
#pragma unroll
    for (int e = 0; e < VPT; ++e) xh.v[e] = xh.v[e] * of.s - of.es;  // past the end not zero, where dy is
    if (PARAMS && live) {
#pragma unroll
      for (int e = 0; e < VPT; ++e) {
        dgamma.v[e] += d.v[e] * xh.v[e];
        dbeta.v[e] += d.v[e];
      }
    }
    if (dx) {
      if (!HOLD) g.load(gamma, cols, lane);
#pragma unroll
      for (int e = 0; e < VPT; ++e) d.v[e] *= g.v[e];
      float a = d.sum(), b = d.dot(xh);
      row_sums<T>(a, b, room[2]);
      a /= n;
      b /= n;
#pragma unroll
      for (int e = 0; e < VPT; ++e) d.v[e] = (d.v[e] - a - xh.v[e] * b) * of.s;
      if (live) d.template store<PAST>(dx + r * cols, cols, lane);
    }
    if (PARAMS) {
      xh = next_x;
      d = next_d;
    }
  }
  if constexpr (PARAMS) {
    if constexpr (ROWS > 1) {
      __shared__ f32x4 sums[ROWS - 1][VPT][T];
      for (int half = 0; half < 2; ++half) {
        Row<T, VPT> &mine = half ? dbeta : dgamma;
        if (half) __syncthreads();
        if (sub > 0) {
#pragma unroll
          for (int e = 0; e < VPT; ++e) sums[sub - 1][e][lane] = mine.v[e];
        }
        __syncthreads();
        if (sub == 0) {
#pragma unroll
          for (int w = 0; w < ROWS - 1; ++w)
#pragma unroll
            for (int e = 0; e < VPT; ++e) mine.v[e] += sums[w][e][lane];
        }
      }
      if (sub > 0) return;
    }
    float *out = partial + (int64_t)blockIdx.x * 2 * padded(cols);
    dgamma.store(out, cols, lane);
    dbeta.store(out + padded(cols), cols, lane);
  }
}

// Long rows: mean, s and es go to `stats`, for the sums over rows that follow.
__global__ __launch_bounds__(kLong) void backward_long_kernel(const float *__restrict__ x, const float *__restrict__ gamma,
                                                             const float *__restrict__ dy, float *__restrict__ dx,
                                                             float *__restrict__ stats, int64_t rows, int cols, float n,
                                                             float eps) {
  __shared__ float rooms[3][kLong / 64][2];
  if (group_index() >= rows) return;
  const int64_t base = group_index() * cols;
  const float *row = x + base, *d = dy + base;
  float mean;
  const Spread of = long_spread(row, cols, n, eps, rooms, mean);
  if (stats && threadIdx.x == 0) {
    float *to = stats + 3 * group_index();
    to[0] = mean;
    to[1] = of.s;
    to[2] = of.es;
  }
  if (!dx) return;
  float sums[2];
  sum_columns(cols, sums, [&](int c, float (&run)[2]) {
    const float t = d[c] * gamma[c];
    run[0] += t;
    run[1] += t * ((row[c] - mean) * of.s - of.es);
  });
  row_sums<kLong>(sums[0], sums[1], rooms[2]);
  const float a = sums[0] / n, b = sums[1] / n;
  for (int c = threadIdx.x; c < cols; c += kLong)
    dx[base + c] = (d[c] * gamma[c] - a - ((row[c] - mean) * of.s - of.es) * b) * of.s;
}

// 64 columns and a run of rows a workgroup; partial as above.
__global__ __launch_bounds__(256) void column_sums_kernel(const float *__restrict__ x, const float *__restrict__ dy,
                                                         const float *__restrict__ stats, float *__restrict__ partial,
                                                         int64_t rows, int cols) {
  __shared__ float sums[2][3][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float dgamma = 0.f, dbeta = 0.f;
  if (c < cols)
    for (int64_t r = (int64_t)blockIdx.y * 4 + wave; r < rows; r += (int64_t)gridDim.y * 4) {
      const float d = dy[r * cols + c];
      dgamma += d * ((x[r * cols + c] - stats[3 * r]) * stats[3 * r + 1] - stats[3 * r + 2]);
      dbeta += d;
    }
  if (wave > 0) {
    sums[0][wave - 1][lane] = dgamma;
    sums[1][wave - 1][lane] = dbeta;
  }
  __syncthreads();
  if (wave > 0 || c >= cols) return;
  for (int w = 0; w < 3; ++w) {
    dgamma += sums[0][w][lane];
    dbeta += sums[1][w][lane];
  }
  float *out = partial + (int64_t)blockIdx.y * 2 * padded(cols);
  out[c] = dgamma;
  out[padded(cols) + c] = dbeta;
}

// dgamma and dbeta from `pieces` partial sums: kSumCols columns of both, one behind the other, a workgroup, and every kSlices-th
// piece a lane, added up in their order.  No pieces (no rows): zeros.  4 096 x 1 024 and 5 003 x 1 537, whole backward pass, with 64 /
// 32 / 16 / 8 columns: 15.7 / 14.5 / 14.7 / 16.1 and 25.4 / 23.8 / 25.1 / 28.0 us.
constexpr int kSlices = 1024 / kSumCols;
__global__ __launch_bounds__(1024) void sum_pieces_kernel(const float *__restrict__ partial, float *__restrict__ dgamma,
                                                         float *__restrict__ dbeta, int pieces, int cols) {
  __shared__ float sums[kSlices][kSumCols];
  const int along = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols;
  const int64_t c = group_index() * kSumCols + along, width = 2 * padded(cols);
  if (c >= width) return;  // the whole workgroup
  float s = 0.f;
  int p = slice;
  for (; p + 3 * kSlices < pieces; p += 4 * kSlices) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = partial[(p + e * kSlices) * width + c];
    s += (v[0] + v[1]) + (v[2] + v[3]);
  }
  for (; p < pieces; p += kSlices) s += partial[p * width + c];
  sums[slice][along] = s;
  __syncthreads();
  if (threadIdx.x >= kSumCols) return;
  for (int w = 1; w < kSlices; ++w) s += sums[w][along];
  float *out = c < width / 2 ? dgamma : dbeta;
  const int64_t to = c < width / 2 ? c : c - width / 2;
  if (out && to < cols) out[to] = s;  // behind the last column there is nothing
}

// x [rows, cols] as the last axis makes it, or an error
int geometry(const char *what, const DLArray *x, const DLArray *gamma, int64_t &rows, int64_t &cols) {
  if (!on_gpu(x) || !on_gpu(gamma)) {
    fprintf(stderr, "[tinyflow_amd] %s: arrays must live on the GPU\n", what);
    return -1;
  }
  if (x->ndim < 1 || gamma->ndim != 1 || gamma->shape[0] != x->shape[x->ndim - 1] || gamma->shape[0] > 1 << 26) {
    fprintf(stderr, "[tinyflow_amd] %s: gamma must hold one value for each column of the last axis (2^26 at most)\n", what);
    return -1;
  }
  cols = gamma->shape[0];
  rows = cols ? numel(x) / cols : 0;
  if (rows > 0x7fffffff) {
    fprintf(stderr, "[tinyflow_amd] %s: 2^31 rows or more are not supported\n", what);
    return -1;
  }
  return 0;
}

// Results of half of what the L2s hold together and more go past them: forward of 8 192 x 2 048 29.2 -> 22.0 us, backward of
// 5 003 x 1 537 22.9 -> 20.4, of 4 096 x 1 024 13.2 -> 11.8; of smaller ones the next reader finds a part, and the writer gains
// nothing (forward of 1 024 x 2 048 4.6 and 4.4).
bool past_caches(int64_t elements) { return elements * 4 >= (int64_t)16 << 20; }

constexpr int kMaxForward = 16384, kMaxBackward = 16384;  // columns that registers hold

}  // namespace

extern "C" int DLGpuLayerNormalizationForward(const DLArrayHandle input, const DLArrayHandle gamma,
                                              const DLArrayHandle beta, DLArrayHandle output, float eps, void **stream) {
  int64_t rows, cols;
  if (geometry(__func__, input, gamma, rows, cols) != 0) return -1;
  TF_REQUIRE(on_gpu(beta) && on_gpu(output), "arrays must live on the GPU");
  TF_REQUIRE(same_shape(beta, gamma), "beta must have gamma's shape");
  TF_REQUIRE(same_shape(input, output), "output must have the input's shape");
  TF_REQUIRE(same_device({input, gamma, beta, output}), "arrays must live on one device");
  TF_REQUIRE(!overlaps(output, gamma) && !overlaps(output, beta), "output must not overlap gamma or beta");
  TF_REQUIRE(input->data == output->data || !overlaps(input, output), "output must be the input or not overlap it");
  TF_REQUIRE(eps >= 0.f, "eps must not be negative");
  announce_write(output);
  hipStream_t s = stream_of(stream);
  if (rows == 0 || cols == 0) return 0;
  const float *x = (const float *)input->data, *g = (const float *)gamma->data, *b = (const float *)beta->data;
  float *y = (float *)output->data;
  const float n = (float)cols;
  auto go = [&](auto t, auto vectors) {
    constexpr int T = decltype(t)::value, VPT = decltype(vectors)::value, WG = T > 256 ? T : 256, ROWS = WG / T;
    hipLaunchKernelGGL((past_caches(rows * cols) ? forward_kernel<T, VPT, true> : forward_kernel<T, VPT, false>),
                       grid_of((rows + ROWS - 1) / ROWS), dim3(WG), 0, s, x, g, b, y, rows, (int)cols, n, eps);
  };
  if (cols <= 256) go(IC<64>{}, IC<1>{});
  else if (cols <= 512) go(IC<64>{}, IC<2>{});
  else if (cols <= 1024) go(IC<256>{}, IC<1>{});
  else if (cols <= 2048) go(IC<256>{}, IC<2>{});
  else if (cols <= 4096) go(IC<256>{}, IC<4>{});
  else if (cols <= 8192) go(IC<1024>{}, IC<2>{});
  else if (cols <= kMaxForward) go(IC<1024>{}, IC<4>{});
  else
    hipLaunchKernelGGL(forward_long_kernel, grid_of(rows), dim3(kLong), 0, s, x, g, b, y, rows, (int)cols, n, eps);
  return finish(s, "DLGpuLayerNormalizationForward");
}

extern "C" int DLGpuLayerNormalizationBackward(const DLArrayHandle input, const DLArrayHandle gamma,
                                               const DLArrayHandle doutput, DLArrayHandle dinput, DLArrayHandle dgamma,
                                               DLArrayHandle dbeta, float eps, int *memorytoSaving, void **stream) {
  int64_t rows, cols;
  if (geometry(__func__, input, gamma, rows, cols) != 0) return -1;
  TF_REQUIRE(on_gpu(doutput) && same_shape(input, doutput), "doutput must live on the GPU and have the input's shape");
  TF_REQUIRE(dinput || dgamma || dbeta, "no gradient is asked for");
  TF_REQUIRE(!dinput || (on_gpu(dinput) && same_shape(input, dinput)), "dinput must live on the GPU and have the input's shape");
  TF_REQUIRE(!dgamma || (on_gpu(dgamma) && same_shape(gamma, dgamma)), "dgamma must live on the GPU and have gamma's shape");
  TF_REQUIRE(!dbeta || (on_gpu(dbeta) && same_shape(gamma, dbeta)), "dbeta must live on the GPU and have gamma's shape");
  TF_REQUIRE(same_device({input, gamma, doutput, dinput, dgamma, dbeta}), "arrays must live on one device");
  for (const DLArray *read : {(const DLArray *)input, (const DLArray *)gamma, (const DLArray *)doutput})
    for (const DLArray *written : {(const DLArray *)dinput, (const DLArray *)dgamma, (const DLArray *)dbeta})
      TF_REQUIRE(!overlaps(read, written), "gradients must not overlap what they are computed from");
  TF_REQUIRE(!overlaps(dinput, dgamma) && !overlaps(dinput, dbeta) && !overlaps(dgamma, dbeta), "gradients must not overlap");
  TF_REQUIRE(eps >= 0.f, "eps must not be negative");
  for (const DLArray *written : {(const DLArray *)dinput, (const DLArray *)dgamma, (const DLArray *)dbeta}) announce_write(written);
  hipStream_t s = stream_of(stream);
  if (cols == 0) return 0;
  const bool params = dgamma || dbeta, in_registers = cols <= kMaxBackward;
  TF_REQUIRE(!params || !being_captured(s), "the gradients of the weights take scratch, which a captured stream cannot give back");

  // How many workgroups share the rows, each with a partial sum of the weights' gradients: two or three a CU, also of short rows, of which
  // eight are resident but have as many more partial sums to write and to add.  us at 1 / 2 / 3 / 4 / 8 a CU: 8 192 x 100 12.2 / 10.6 /
  // 10.7 / 11.4 / 13.5, x 512 15.4 / 14.3 / 13.7 / 15.3 / 19.4, x 1 024 24.8 / 21.7 / 21.6 / 24.8 / 29.2, x 2 048 47 / 37.2 / 37.4 / 39.6 /
  // 43.8, x 4 096 90 / 71 / 81 / 79 / 93; 50 000 x 256 46 / 31.5 / 30.9 / 31.0 / 33.8, x 1 024 112 / 115 / 118 / 120 / 121, x 2 048 290 / 225 /
  // 237 / 242 / 238, x 4 096 533 / 450 / 497 / 453 / 470; 2 048 rows of up to 1 024 the same within 5 %.  Of more than 4 096 columns a
  // workgroup has 1 024 lanes, of which a CU holds one.
  const int rows_a_group = !in_registers ? 1 : cols <= 1024 ? 4 : cols <= 2048 ? 2 : 1;
  const int64_t groups = (rows + rows_a_group - 1) / rows_a_group;
  int pieces = 0;
  if (in_registers) pieces = (int)std::min<int64_t>(groups, params ? (cols <= 1024 ? 2 : cols <= 2048 ? 3 : cols <= 4096 ? 2 : 1) * num_cus() : 1 << 20);
  else if (rows) pieces = (int)std::min<int64_t>((rows + 3) / 4, std::max<int64_t>(1, 4 * num_cus() * 64 / cols));
  float *partial = nullptr, *stats = nullptr;
  if (params && rows) {
    const size_t partial_bytes = (size_t)pieces * 2 * padded(cols) * 4, stats_bytes = in_registers ? 0 : (size_t)rows * 12;
    partial = (float *)device_alloc(partial_bytes + stats_bytes, s);
    if (!partial) {
      if (memorytoSaving) *memorytoSaving = shortfall(block_bytes(partial_bytes + stats_bytes));
      return 0;
    }
    if (stats_bytes) stats = partial + (size_t)pieces * 2 * padded(cols);
  }
  const float *x = (const float *)input->data, *g = (const float *)gamma->data, *dy = (const float *)doutput->data;
  float *dx = dinput ? (float *)dinput->data : nullptr;
  const float n = (float)cols;
  if (rows) {
    auto go = [&](auto t, auto vectors) {
      constexpr int T = decltype(t)::value, VPT = decltype(vectors)::value, WG = T > 256 ? T : 256;
      const bool past = past_caches(rows * cols);
      hipLaunchKernelGGL((params ? past ? backward_kernel<T, VPT, WG, true, true> : backward_kernel<T, VPT, WG, true, false>
                                 : past ? backward_kernel<T, VPT, WG, false, true> : backward_kernel<T, VPT, WG, false, false>),
                         dim3((unsigned)pieces), dim3(WG), 0, s, x, g, dy, dx, partial, rows, (int)cols, n, eps);
    };
    if (cols <= 256) go(IC<64>{}, IC<1>{});
    else if (cols <= 512) go(IC<64>{}, IC<2>{});
    else if (cols <= 1024) go(IC<64>{}, IC<4>{});
    else if (cols <= 2048) go(IC<128>{}, IC<4>{});
    else if (cols <= 4096) go(IC<512>{}, IC<2>{});
    else if (cols <= 8192) go(IC<1024>{}, IC<2>{});
    else if (in_registers) go(IC<1024>{}, IC<4>{});
    else {
      hipLaunchKernelGGL(backward_long_kernel, grid_of(rows), dim3(kLong), 0, s, x, g, dy, dx, stats, rows, (int)cols, n, eps);
      if (params)
        hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((cols + 63) / 64), (unsigned)pieces), dim3(256), 0, s, x, dy,
                           stats, partial, rows, (int)cols);
    }
  }
  if (params)
    hipLaunchKernelGGL(sum_pieces_kernel, grid_of(2 * padded(cols) / kSumCols), dim3(1024), 0, s, partial,
                       dgamma ? (float *)dgamma->data : nullptr, dbeta ? (float *)dbeta->data : nullptr, rows ? pieces : 0,
                       (int)cols);
  if (partial) device_free(partial, s);
  return finish(s, "DLGpuLayerNormalizationBackward");
}
