// Attention, forward and backward (no counterpart in the reference).  attention.h has the formulas and what rows are.
//
// Forms of the forward pass (which one runs: DLGpuAttentionForward, pair_suits):
//   few_kernel     up to 32 rows of a key head: every wave streams its own keys from memory to registers, nothing is staged; bound by HBM: 100 003 keys of 2
//                  heads of 128, 205 MB, 39 us, 5.2 TB/s
//   rows_kernel    128 rows a workgroup, the fp32 matrix instruction, which bounds it: 4 096 causal tokens of 16 heads on 4 of 128, 69 GFLOP, 1.09 ms
//   attention_pair.hip    the same rows on fp16 pairs, 0.2 ms; rows_kernel then takes what cannot be split
// Both can be cut along the keys: pieces write their unnormalised sums with their maximum, join_kernel adds them up in their order.
// Backward: prepare_kernel (delta, what each row sees), dq_kernel (128 rows a workgroup, walks the keys), dkv_kernel (128 keys a workgroup, walks the
// rows); where that leaves CUs without work the walks are cut, and sum_kernel adds the pieces.  Both compute the scores again; no sum goes
// through atomics, so the bits do not depend on the order in which workgroups run.
#include "attention.h"
#include "few_rows.h"
#include "internal.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

using namespace tf;
using namespace tf::attention;

namespace {

template <int V>
using IC = std::integral_constant<int, V>;

// ------------------------------------------------------------------------------ tiles of the fp32 instruction
//
// v_mfma_f32_32x32x2: a lane supplies A[lane % 32][half] and B[half][lane % 32], half = lane / 32, and holds D[8 (v / 4) + 4 half + v % 4][lane % 32].
// A score tile is computed with what the lane keeps on the columns: rows in the forward pass and dq, keys in dkv.  Its 16 values are then, as they
// are, the B operands of the products that follow: step v takes row 8 (v / 4) + 4 half + v % 4 of the tile on the other side.

// 32 rows of DP columns in LDS, columns past `dim` and rows past `count` zero.  Four floats more than a row keep the reads apart.
template <int DP>
struct Tile {
  static constexpr int LD = DP + 4;
  float v[32][LD];

  // rows of `at(r)`; CLEAN: what is not finite becomes 0, and its row's bit is set in `found`
  template <class At>
  __device__ inline void stage(const At &at, int count, int dim, bool clean, uint32_t *found) {
    constexpr int A_ROW = DP / 4;
#pragma unroll 4
    for (int e = threadIdx.x; e < 32 * A_ROW; e += kThreads) {
      const int r = e / A_ROW, c = e % A_ROW * 4;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (r < count && c < dim) x = load4(at(r) + c, dim - c);
      if (clean) {
        bool all = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool ok = finite(x[i]);
          all &= ok;
          if (!ok) x[i] = 0.f;
        }
        if (!all) atomicOr(found, 1u << r);
      }
      *reinterpret_cast<f32x4 *>(&v[r][c]) = x;
    }
  }
};

// The B operand of a product over columns: of the lane's row or key, columns 8 g + 4 half + e.
template <int DP>
struct Operand {
  f32x4 v[DP / 8];
  __device__ inline void load(const float *row, int dim, bool live) {
    const int half = threadIdx.x % 64 / 32;
#pragma unroll
    for (int g = 0; g < DP / 8; ++g) {
      const int c = 8 * g + 4 * half;
      v[g] = live && c < dim ? load4(row + c, dim - c) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  __device__ inline float dot(const Operand &o) const {  // over all columns
    f32x4 s = v[0] * o.v[0];
#pragma unroll
    for (int g = 1; g < DP / 8; ++g) s += v[g] * o.v[g];
    const float t = (s[0] + s[1]) + (s[2] + s[3]);
    return t + other_half(t);
  }
};

template <int DP>
__device__ inline f32x16 scores(const Tile<DP> &a, const Operand<DP> &b) {
  const int half = threadIdx.x % 64 / 32, row = threadIdx.x % 32;
  f32x16 s;
#pragma unroll
  for (int v = 0; v < 16; ++v) s[v] = 0.f;
#pragma unroll
  for (int g = 0; g < DP / 8; ++g) {
    const f32x4 x = *reinterpret_cast<const f32x4 *>(&a.v[row][8 * g + 4 * half]);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], b.v[g][e], s, 0, 0, 0);
  }
  return s;
}

// What staging took out of the tile, in the products again: those of rows `found`, from the operands as they were.
template <int DP, class At>
__device__ inline void repair(f32x16 &s, uint32_t found, const At &at, int dim, const Operand<DP> &b) {
  const int half = threadIdx.x % 64 / 32;
#pragma unroll 1
  for (; found; found &= found - 1) {
    const int r = __builtin_ctz(found), from = r / 4 % 2, e = r / 8 * 4 + r % 4;
    Operand<DP> a;
    a.load(at(r), dim, true);
    const float x = a.dot(b);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = i == e && from == half ? x : s[i];
  }
}

// sum[block][v] += of column 32 block + key_of(v, half), over the tile's rows with the lane's weights
template <int DP>
struct Sum {
  f32x16 v[DP / 32];
  __device__ inline void zero() {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) v[d][e] = 0.f;
  }
  __device__ inline void add(const Tile<DP> &a, const float (&w)[16]) {
    const int half = threadIdx.x % 64 / 32, col = threadIdx.x % 32;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        v[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[key_of(e, half)][32 * d + col], w[e], v[d], 0, 0, 0);
  }
  // What staging took out of the tile, back with the weights that are not 0: rows `found`, read again at `at(row)`.
  template <class At>
  __device__ inline void add_back(uint32_t found, const At &at, int dim, const float (&w)[16]) {
    const int half = threadIdx.x % 64 / 32;
#pragma unroll 1
    for (; found; found &= found - 1) {
      const int r = __builtin_ctz(found), from = r / 4 % 2, e = r / 8 * 4 + r % 4;
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) x = i == e ? w[i] : x;
      const float weight = __shfl(x, threadIdx.x % 32 + 32 * from);
      const float *row = at(r);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = 32 * d + key_of(i, half);
          if (c < dim && !finite(row[c]) && weight != 0.f) v[d][i] += weight * row[c];
        }
    }
  }
  __device__ inline void scale(float by) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) v[d] *= by;
  }
};

// ------------------------------------------------------------------------------ forward, 128 rows a workgroup

template <int DP>
__global__ __launch_bounds__(kThreads) void rows_kernel(const Call c, float *out, float *stat, const Pieces pieces, int tiles,
                                                        const Exponents left) {
  __shared__ __align__(16) Tile<DP> kt, vt;
  __shared__ int room[4][4];
  __shared__ uint32_t found;
  const int bg = (int)blockIdx.x % (c.batch * c.key_heads), rest = (int)blockIdx.x / (c.batch * c.key_heads);
  const int b = bg / c.key_heads, g = bg % c.key_heads, tile = tiles - 1 - rest % tiles, piece = rest / tiles;
  if (left.q && !__syncthreads_or(left.bad_head(bg))) return;
  const int lane = threadIdx.x % 64, half = lane / 32;
  const int r = tile * kRows + threadIdx.x / 64 * 32 + lane % 32;
  const bool live = r < c.rows;
  const int i = (live ? r : c.rows - 1) / c.group;
  int lo, hi, at;
  c.seen(b, i, lo, hi, at);
  const int near = c.nearest(at, lo, hi);
  const float slope = c.slopes ? c.slopes[g * c.group + (live ? r : 0) % c.group] * kLog2e : 0.f;
  Hull mine;
  mine.of(lo, hi, live);
  const Hull all = mine.all(room);
  // this piece's steps of the keys that any of the rows sees
  const int first = all.first(), steps = all.steps();
  if (left.q && !__syncthreads_or(left.bad_rows(bg, tile * (kRows / 32), first, steps))) return;
  Operand<DP> q;
  q.load(c.q + c.query_at(b, g, live ? r : 0), c.dim, live);
  const int begin = first + (int)((int64_t)steps * piece / pieces.count), end = first + (int)((int64_t)steps * (piece + 1) / pieces.count);
  const Score score(c);
  Sum<DP> o;
  o.zero();
  float top = kNone, total = 0.f;
#pragma unroll 1
  for (int step = begin; step < end; ++step) {
    const int j0 = step * kKeys, count = min(kKeys, c.tk - j0);
    const bool clean = !all.covers(j0, j0 + kKeys);
    __syncthreads();
    if (threadIdx.x == 0) found = 0u;
    if (clean) __syncthreads();
    kt.stage([&](int n) { return c.k + c.key_at(b, g, j0 + n); }, count, c.dim, false, nullptr);
    vt.stage([&](int n) { return c.v + c.key_at(b, g, j0 + n); }, count, c.dim, clean, &found);
    __syncthreads();
    if (!mine.meets(j0, j0 + kKeys)) continue;
    const f32x16 s = scores(kt, q);
    float p[16], most = kNone;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int j = j0 + key_of(v, half);
      p[v] = score(s[v]) - slope * fabsf((float)(near - j));
      if (!mine.covers(j0, j0 + kKeys)) p[v] = j >= lo && j < hi ? p[v] : kNone;
      most = fmaxf(most, p[v]);
    }
    most = fmaxf(most, other_half(most));
    const float next = fmaxf(top, most), from = next == kNone ? 0.f : next;
    const float fade = __builtin_amdgcn_exp2f(top - from);
    top = next;
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      p[v] = __builtin_amdgcn_exp2f(p[v] - from);
      sum += p[v];
    }
    total = total * fade + (sum + other_half(sum));
    if (__any(fade != 1.f)) o.scale(fade);
    o.add(vt, p);
    if (clean && found) o.add_back(found, [&](int n) { return c.v + c.key_at(b, g, j0 + n); }, c.dim, p);
  }
  if (!live) return;
  float *row;
  const float by = row_end(c, pieces, out, stat, b, g, r, piece, top, total, half == 0, row);
  if (row) store_sums(o.v, row, c.dim, by);
}

// ------------------------------------------------------------------------------ forward, few rows

// v_mfma_f32_16x16x4: a lane supplies A[lane % 16][lane / 16] and B[lane / 16][lane % 16] and holds D[4 (lane / 16) + v][lane % 16].  Scores: keys by
// rows, columns 16 g + 4 (lane / 16) + e of both.  The values' product takes key 4 (lane / 16) + v at step v, as the scores lie,
// and sums column 64 d + 4 (row of D) + e into sum[d][e]: both operands are 16-byte loads from where they lie in memory, 16 lanes side by side.
// What bounds it is HBM as long as a wave's next step is on its way all the time that one is worked on: with the next keys fetched behind the
// scores and the next values behind their product, and loads behind branches, of which all are waited for, 100 003 keys of 2 heads of 128 took 49 us,
// and so 39-41 (5.0-5.2 TB/s).
constexpr int kFewKeys = 16;  // of a wave's step

// op over the four lanes with the same lane % 16
template <class Op>
__device__ inline float over_quarters(float v, const Op &op) {
  uint32_t bits = __builtin_bit_cast(uint32_t, v);
  auto halves = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
  v = op(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
  bits = __builtin_bit_cast(uint32_t, v);
  halves = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
  return op(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}

template <int DP, int NC>
__global__ __launch_bounds__(kThreads, DP * NC <= 128 ? 2 : 1) void few_kernel(const Call c, float *out, float *stat, const Pieces pieces, int keys_a_piece) {
  constexpr int GD = DP / 16, VD = DP / 64;
  const int bg = (int)blockIdx.x % (c.batch * c.key_heads), piece = (int)blockIdx.x / (c.batch * c.key_heads);
  const int b = bg / c.key_heads, g = bg % c.key_heads;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, quarter = lane / 16, col = lane % 16;
  int lo[NC], hi[NC], near[NC], all_lo = INT32_MAX, all_hi = 0, inner_lo = 0, inner_hi = INT32_MAX;
  float slope[NC];
  f32x4 q[NC][GD];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int r = 16 * n + col;
    const bool live = r < c.rows;
    const int i = (live ? r : 0) / c.group;
    int at;
    c.seen(b, i, lo[n], hi[n], at);
    near[n] = c.nearest(at, lo[n], hi[n]);
    if (!live) hi[n] = 0;
    slope[n] = c.slopes && live ? c.slopes[g * c.group + r % c.group] * kLog2e : 0.f;
    const float *row = c.q + c.query_at(b, g, live ? r : 0);
#pragma unroll
    for (int e = 0; e < GD; ++e) {
      const int d = 16 * e + 4 * quarter;
      q[n][e] = live && d < c.dim ? load4(row + d, c.dim - d) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (lo[n] < hi[n]) {
      all_lo = min(all_lo, lo[n]);
      all_hi = max(all_hi, hi[n]);
    }
    if (live) {  // columns that are no rows may hold anything
      inner_lo = max(inner_lo, lo[n]);
      inner_hi = min(inner_hi, hi[n]);
    }
  }
#pragma unroll
  for (int step = 1; step < 16; step *= 2) {
    all_lo = min(all_lo, __shfl_xor(all_lo, step));
    all_hi = max(all_hi, __shfl_xor(all_hi, step));
    inner_lo = max(inner_lo, __shfl_xor(inner_lo, step));
    inner_hi = min(inner_hi, __shfl_xor(inner_hi, step));
  }
  if (all_lo >= all_hi) all_lo = all_hi = 0;  // nothing is seen
  const int begin = max(__builtin_amdgcn_readfirstlane(all_lo) / kFewKeys * kFewKeys, piece * keys_a_piece);
  const int end = min(__builtin_amdgcn_readfirstlane(all_hi), (piece + 1) * keys_a_piece);  // a piece is a multiple of 64 keys
  inner_lo = __builtin_amdgcn_readfirstlane(inner_lo);
  inner_hi = __builtin_amdgcn_readfirstlane(inner_hi);

  const Score score(c);
  f32x4 o[NC][VD][4];
  float top[NC], total[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    top[n] = kNone;
    total[n] = 0.f;
#pragma unroll
    for (int d = 0; d < VD; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][d][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int64_t key_step = (int64_t)c.key_heads * c.dim;
  const float *k0 = c.k + c.key_at(b, g, 0), *v0 = c.v + c.key_at(b, g, 0);
  // Loads without a branch, so that it is known how many are under way: columns that are none have an offset behind the buffer and read as zero, and
  // keys behind the last are the last again.  The buffer ends with the array: four columns of a head whose length is no multiple of four may reach
  // behind the last one.
  typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u32x4;
  f32x4 keys[2][GD], values[2][4][VD];
  const int64_t in_array = (int64_t)c.batch * c.tk * key_step, head_at = c.key_at(b, g, 0);
  int bytes;
  auto fetch = [&](const float *base, int row, int column) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(base), 0, bytes, 0x00020000);
    f32x4 x = __builtin_bit_cast(f32x4, (u32x4)__builtin_amdgcn_raw_buffer_load_b128(r, (int)buffer_offset(row, key_step, column, c.dim), 0, 0));
    return x;
  };
  auto load = [&](auto parity, int j0) {
    j0 = __builtin_amdgcn_readfirstlane(min(j0, end - 1));
    const float *kb = k0 + j0 * key_step, *vb = v0 + j0 * key_step;
    bytes = buffer_bytes(in_array, head_at + j0 * key_step);
    const int last = end - 1 - j0;
#pragma unroll
    for (int e = 0; e < GD; ++e) keys[decltype(parity)::value][e] = fetch(kb, min(col, last), 16 * e + 4 * quarter);
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int d = 0; d < VD; ++d) values[decltype(parity)::value][v][d] = fetch(vb, min(4 * quarter + v, last), 64 * d + 4 * col);
  };
  // rows whose length is no multiple of four: what a load brought from behind their end
  auto cut = [&](f32x4 &x, int column) {
#pragma unroll
    for (int i = 1; i < 4; ++i) x[i] = column + i < c.dim ? x[i] : 0.f;
  };
  auto step = [&](auto parity, int j0) {
    auto &k = keys[decltype(parity)::value];
    auto &vals = values[decltype(parity)::value];
    if (c.dim % 4) {
#pragma unroll
      for (int e = 0; e < GD; ++e) cut(k[e], 16 * e + 4 * quarter);
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int d = 0; d < VD; ++d) cut(vals[v][d], 64 * d + 4 * col);
    }
    const bool whole = inner_lo <= j0 && inner_hi >= j0 + kFewKeys && end >= j0 + kFewKeys;
    float p[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < GD; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e][x], q[n][e][x], s, 0, 0, 0);
      float most = kNone;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int j = j0 + 4 * quarter + v;
        p[n][v] = score(s[v]) - slope[n] * fabsf((float)(near[n] - j));
        if (!whole) p[n][v] = j >= lo[n] && j < hi[n] && j < end ? p[n][v] : kNone;
        most = fmaxf(most, p[n][v]);
      }
      most = over_quarters(most, [](float a, float b) { return fmaxf(a, b); });
      const float next = fmaxf(top[n], most), from = next == kNone ? 0.f : next;
      const float fade = __builtin_amdgcn_exp2f(top[n] - from);
      top[n] = next;
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        p[n][v] = __builtin_amdgcn_exp2f(p[n][v] - from);
        sum += p[n][v];
      }
      total[n] = total[n] * fade + sum;  // of this lane's keys
      if (__any(fade != 1.f)) {
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][d][e] *= fade;
      }
    }
    if (!whole) {
      // values that are not finite: only to the rows that see them
      bool ok = true;
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) ok &= finite(vals[v][d][e]);
      if (__any(!ok)) {
#pragma unroll 1
        for (int t = 0; t < kFewKeys; ++t) {
          const float *row = v0 + (int64_t)min(j0 + t, end - 1) * key_step;
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            float w = 0.f;
#pragma unroll
            for (int v = 0; v < 4; ++v) w = t % 4 == v ? p[n][v] : w;
            w = __shfl(w, col + t / 4 * 16);
#pragma unroll
            for (int d = 0; d < VD; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  const int at = 64 * d + 16 * quarter + 4 * v + e;
                  if (at < c.dim && w != 0.f && !finite(row[at])) o[n][d][e][v] += w * row[at];
                }
          }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int d = 0; d < VD; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) vals[v][d][e] = finite(vals[v][d][e]) ? vals[v][d][e] : 0.f;
      }
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][d][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vals[v][d][e], p[n][v], o[n][d][e], 0, 0, 0);
  };
  constexpr int STEP = 4 * kFewKeys;
  int j0 = begin + kFewKeys * wave;
  if (j0 < end) load(IC<0>{}, j0);
#pragma unroll 1
  for (; j0 < end; j0 += 2 * STEP) {
    load(IC<1>{}, j0 + STEP);
    step(IC<0>{}, j0);
    if (j0 + STEP >= end) break;
    load(IC<0>{}, j0 + 2 * STEP);
    step(IC<1>{}, j0 + STEP);
  }

  // the four waves' sums, through LDS in their order
  __shared__ float marks[4][16][2];
  __shared__ f32x4 parts[3][VD * 4][64];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    total[n] = over_quarters(total[n], [](float a, float b) { return a + b; });
    if (n) __syncthreads();
    if (quarter == 0) {
      marks[wave][col][0] = top[n];
      marks[wave][col][1] = total[n];
    }
    __syncthreads();
    float most = kNone, whole = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) most = fmaxf(most, marks[w][col][0]);
    const float from = most == kNone ? 0.f : most;
#pragma unroll
    for (int w = 0; w < 4; ++w) whole += marks[w][col][1] * __builtin_amdgcn_exp2f(marks[w][col][0] - from);
    const float fade = __builtin_amdgcn_exp2f(top[n] - from);
#pragma unroll
    for (int d = 0; d < VD; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[n][d][e] *= fade;
        if (wave > 0) parts[wave - 1][d * 4 + e][lane] = o[n][d][e];
      }
    __syncthreads();
    const int r = 16 * n + col;
    if (wave == 0 && r < c.rows) {
      float *row;
      const float by = row_end(c, pieces, out, stat, b, g, r, piece, most, whole, quarter == 0, row);
#pragma unroll
      for (int d = 0; d < VD; ++d) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int w = 0; w < 3; ++w) o[n][d][e] += parts[w][d * 4 + e][lane];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int at = 64 * d + 16 * quarter + 4 * v;
          if (row && at < c.dim) store4(row + at, c.dim - at, f32x4{o[n][d][0][v] * by, o[n][d][1][v] * by, o[n][d][2][v] * by, o[n][d][3][v] * by});
        }
      }
    }
  }
}

// Rows of all from their pieces, in the pieces' order: a row to W waves, each with a run of the pieces.  The pieces' factors are in LDS before their
// sums are read, eight loads of a lane under way: with each sum behind the branch on its mark 512 pieces of 16 rows of 128 took 44 us.
constexpr int kMostPieces = 2048;
template <int W>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void join_kernel(const Call c, const Pieces pieces, float *out, float *stat) {
  constexpr int ROWS = W > 4 ? 1 : 4 / W, LANES = 64 * W, MOST = 4, UNDER_WAY = 8;  // MOST: columns of a lane
  __shared__ float by[ROWS][W > 1 ? kMostPieces : 16];
  __shared__ float parts[W > 1 ? W : 1][MOST][64];
  __shared__ float tops[W], totals[W];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, sub = wave % W, own = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * ROWS + wave / W;
  if (row >= pieces.rows) return;  // with one wave a row
  float *const weights = by[wave / W];
  float top = kNone, total = 0.f;
  for (int p = own; p < pieces.count; p += LANES) top = fmaxf(top, pieces.marks[p * pieces.rows + row].x);
#pragma unroll
  for (int step = 1; step < 64; step *= 2) top = fmaxf(top, __shfl_xor(top, step));
  if constexpr (W > 1) {
    if (lane == 0) tops[sub] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, tops[w]);
  }
  const float from = top == kNone ? 0.f : top;
  for (int p = own; p < pieces.count; p += LANES) {
    const float2 mark = pieces.marks[p * pieces.rows + row];
    const float factor = __builtin_amdgcn_exp2f(mark.x - from);
    total += mark.y * factor;
    weights[p] = mark.y == 0.f ? 0.f : factor;  // nothing seen: nothing stored that counts
  }
#pragma unroll
  for (int step = 1; step < 64; step *= 2) total += __shfl_xor(total, step);
  if constexpr (W > 1) {
    if (lane == 0) totals[sub] = total;
    __syncthreads();
    total = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) total += totals[w];
  } else {
    __builtin_amdgcn_wave_barrier();
  }
  const int each = (pieces.count + W - 1) / W, begin = min(pieces.count, sub * each), end = min(pieces.count, begin + each);
  float sum[MOST] = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = begin; p0 < end; p0 += UNDER_WAY) {
#pragma unroll
    for (int e = 0; e < MOST; ++e) {
      if (64 * e >= c.dim) break;
      float v[UNDER_WAY];
#pragma unroll
      for (int u = 0; u < UNDER_WAY; ++u)
        v[u] = pieces.sums[((int64_t)min(p0 + u, end - 1) * pieces.rows + row) * c.dim + min(lane + 64 * e, c.dim - 1)];
#pragma unroll
      for (int u = 0; u < UNDER_WAY; ++u) {
        const float factor = p0 + u < end ? weights[p0 + u] : 0.f;
        sum[e] += factor != 0.f ? v[u] * factor : 0.f;
      }
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < MOST; ++e) parts[sub][e][lane] = sum[e];
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int e = 0; e < MOST; ++e)
      for (int w = 1; w < W; ++w) sum[e] += parts[w][e][lane];
  }
  const int r = (int)(row % c.rows), g = (int)(row / c.rows % c.key_heads), b = (int)(row / c.rows / c.key_heads);
  if (stat && lane == 0) stat[c.stat_at(b, g, r)] = total == 0.f ? kNone : c.statistic(b, g, r, top + __builtin_amdgcn_logf(total));
  if (!out) return;
  const float scale = total == 0.f ? 0.f : 1.f / total;
  float *to = out + c.query_at(b, g, r);
#pragma unroll
  for (int e = 0; e < MOST; ++e)
    if (lane + 64 * e < c.dim) to[lane + 64 * e] = sum[e] * scale;
}

// ------------------------------------------------------------------------------ backward

// A wave a row of all.
__global__ __launch_bounds__(kThreads) void prepare_kernel(const Call c, const float *__restrict__ o, const float *__restrict__ stat,
                                                           const float *__restrict__ dout, Row *__restrict__ rows, int64_t count) {
  const int64_t at = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (at >= count) return;
  const int r = (int)(at % c.rows), g = (int)(at / c.rows % c.key_heads), b = (int)(at / c.rows / c.key_heads), lane = threadIdx.x % 64;
  const int64_t from = c.query_at(b, g, r);
  float delta = 0.f;
  for (int d = lane; d < c.dim; d += 64) delta += o[from + d] * dout[from + d];
#pragma unroll
  for (int step = 1; step < 64; step *= 2) delta += __shfl_xor(delta, step);
  if (lane > 0) return;
  Row row;
  c.seen(b, r / c.group, row.lo, row.hi);
  row.stat = c.taken(b, g, r, row.lo, row.hi, stat[c.stat_at(b, g, r)]);
  row.delta = delta;
  if (row.lo >= row.hi || row.stat == kNone) row.lo = row.hi = 0;
  rows[at] = row;
}

// 128 rows a workgroup, 32 a wave, and of the keys that they see piece blockIdx.x / (tiles * heads); a piece's results are `stride` behind the one's before.
template <int DP>
__global__ __launch_bounds__(kThreads) void dq_kernel(const Call c, const float *dout, const Row *rows, float *dq, int64_t stride, int tiles, int pieces, const Exponents left) {
  __shared__ __align__(16) Tile<DP> kt, vt;
  __shared__ int room[4][4];
  __shared__ uint32_t found;
  const int bg = (int)blockIdx.x % (c.batch * c.key_heads), rest = (int)blockIdx.x / (c.batch * c.key_heads);
  const int b = bg / c.key_heads, g = bg % c.key_heads, tile = tiles - 1 - rest % tiles, piece = rest / tiles;
  if (left.q && !__syncthreads_or(left.bad_head(bg))) return;
  const int lane = threadIdx.x % 64, half = lane / 32;
  const int r = tile * kRows + threadIdx.x / 64 * 32 + lane % 32;
  const bool live = r < c.rows;
  const Row row = rows[(int64_t)bg * c.rows + (live ? r : 0)];
  const int near = c.nearest(c.own(b, (live ? r : 0) / c.group), row.lo, row.hi);
  const float slope = c.slopes ? c.slopes[g * c.group + (live ? r : 0) % c.group] * kLog2e : 0.f;
  const int64_t at = c.query_at(b, g, live ? r : 0);
  Hull mine;
  mine.of(row.lo, row.hi, live);
  const Hull all = mine.all(room);
  const int first = all.first(), steps = all.steps();
  if (left.q && !__syncthreads_or(left.bad_rows(bg, tile * (kRows / 32), first, steps))) return;
  const int begin = first + (int)((int64_t)steps * piece / pieces), end = first + (int)((int64_t)steps * (piece + 1) / pieces);
  Operand<DP> q, d;
  q.load(c.q + at, c.dim, live);
  d.load(dout + at, c.dim, live);
  const Score score(c);
  Sum<DP> sum;
  sum.zero();
#pragma unroll 1
  for (int step = begin; step < end; ++step) {
    const int j0 = step * kKeys, count = min(kKeys, c.tk - j0);
    const bool clean = !all.covers(j0, j0 + kKeys);
    __syncthreads();
    if (threadIdx.x == 0) found = 0u;
    if (clean) __syncthreads();
    kt.stage([&](int n) { return c.k + c.key_at(b, g, j0 + n); }, count, c.dim, clean, &found);
    vt.stage([&](int n) { return c.v + c.key_at(b, g, j0 + n); }, count, c.dim, false, nullptr);
    __syncthreads();
    if (!mine.meets(j0, j0 + kKeys)) continue;
    f32x16 s = scores(kt, q);
    if (clean && found) repair(s, found, [&](int n) { return c.k + c.key_at(b, g, j0 + n); }, c.dim, q);
    const f32x16 dp = scores(vt, d);
    float ds[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int j = j0 + key_of(v, half);
      float p;
      gradient(score, s[v], dp[v], slope * fabsf((float)(near - j)), row.stat, row.delta, j >= row.lo && j < row.hi, p, ds[v]);
    }
    sum.add(kt, ds);
    if (clean && found) sum.add_back(found, [&](int n) { return c.k + c.key_at(b, g, j0 + n); }, c.dim, ds);
  }
  if (live) store_sums(sum.v, dq + piece * stride + at, c.dim, c.scale);
}

// 128 keys a workgroup, 32 a wave, which walks the rows of piece blockIdx.x / (tiles * heads).  Results go to dk and dv, or piece by piece to
// [piece][2][b, key, key head][dim].
template <int DP, bool DK, bool DV>
__global__ __launch_bounds__(kThreads) void dkv_kernel(const Call c, const float *dout, const Row *rows, float *dk, float *dv, float *parts,
                                                       int tiles, int pieces, const Exponents left) {
  __shared__ __align__(16) Tile<DP> qt, dt;
  __shared__ Row info[32];
  __shared__ float slopes[32];
  __shared__ int nears[32];
  __shared__ int meet[3];  // least and greatest key that a row of the step sees, whether any sees less than all of the tile
  __shared__ uint32_t found_q, found_d;
  const int bg = (int)blockIdx.x % (c.batch * c.key_heads), rest = (int)blockIdx.x / (c.batch * c.key_heads);
  const int b = bg / c.key_heads, g = bg % c.key_heads, tile = rest % tiles, piece = rest / tiles;
  const int lane = threadIdx.x % 64, half = lane / 32;
  const int tile_lo = tile * kRows, tile_hi = min(c.tk, tile_lo + kRows);
  const int j = tile_lo + threadIdx.x / 64 * 32 + lane % 32;
  if (left.q && !__syncthreads_or(left.bad_keys(bg, tile_lo / 32, tile_lo, tile_hi))) return;
  const bool live = j < c.tk;
  const int64_t at = c.key_at(b, g, live ? j : 0);
  Operand<DP> k, v;
  k.load(c.k + at, c.dim, live);
  if (DK) v.load(c.v + at, c.dim, live);
  const Score score(c);
  Sum<DP> dks, dvs;
  if (DK) dks.zero();
  if (DV) dvs.zero();
  const int steps = (c.rows + 31) / 32;
  const int begin = (int)((int64_t)steps * piece / pieces), end = (int)((int64_t)steps * (piece + 1) / pieces);
  const Row *of = rows + (int64_t)bg * c.rows;
#pragma unroll 1
  for (int step = begin; step < end; ++step) {
    const int r0 = step * 32, count = min(32, c.rows - r0);
    __syncthreads();
    if (threadIdx.x < 64) {
      const int r = r0 + threadIdx.x;
      const bool is = threadIdx.x < (unsigned)count;
      Row row = {0.f, 0.f, 0, 0};
      if (is) row = of[r];
      if (threadIdx.x < 32) {
        info[threadIdx.x] = row;
        nears[threadIdx.x] = is ? c.nearest(c.own(b, r / c.group), row.lo, row.hi) : 0;
        slopes[threadIdx.x] = c.slopes && is ? c.slopes[g * c.group + r % c.group] * kLog2e : 0.f;
      }
      const bool sees = is && row.lo < tile_hi && row.hi > tile_lo;
      const bool any = __any(sees), part = __any(threadIdx.x < 32 && !(is && row.lo <= tile_lo && row.hi >= tile_lo + kRows));
      if (threadIdx.x == 0) {
        meet[0] = any;
        meet[1] = part;
        found_q = found_d = 0u;
      }
    }
    __syncthreads();
    if (!meet[0]) continue;
    const bool clean = meet[1] != 0;
    auto q_at = [&](int n) { return c.q + c.query_at(b, g, r0 + n); };
    auto d_at = [&](int n) { return dout + c.query_at(b, g, r0 + n); };
    qt.stage(q_at, count, c.dim, clean && DK, &found_q);
    dt.stage(d_at, count, c.dim, clean && DV, &found_d);
    __syncthreads();
    f32x16 s = scores(qt, k), dp = s;
    if (DK) dp = scores(dt, v);
    if (clean && DK && found_q) repair(s, found_q, q_at, c.dim, k);
    if (clean && DK && DV && found_d) repair(dp, found_d, d_at, c.dim, v);
    float p[16], ds[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int n = key_of(e, half);
      const Row row = info[n];
      const float bias = slopes[n] * fabsf((float)(nears[n] - j));
      gradient(score, s[e], dp[e], bias, row.stat, row.delta, live && j >= row.lo && j < row.hi, p[e], ds[e]);
    }
    if (DV) {
      dvs.add(dt, p);
      if (clean && found_d) dvs.add_back(found_d, d_at, c.dim, p);
    }
    if (DK) {
      dks.add(qt, ds);
      if (clean && found_q) dks.add_back(found_q, q_at, c.dim, ds);
    }
  }
  if (!live) return;
  const int64_t all = (int64_t)c.batch * c.tk * c.key_heads * c.dim;
  if (DK) store_sums(dks.v, (pieces > 1 ? parts + (int64_t)piece * 2 * all : dk) + at, c.dim, c.scale);
  if (DV) store_sums(dvs.v, (pieces > 1 ? parts + ((int64_t)piece * 2 + 1) * all : dv) + at, c.dim, 1.f);
}

// Gradients from their pieces, in order: blockIdx.y says which, `stride` is from one piece to the next.
struct Job {
  const float *from;
  float *to;
  int64_t all, stride;
  int pieces;
};
struct Jobs {
  Job job[3];
  int n;
};
__global__ __launch_bounds__(kThreads) void sum_kernel(const Jobs jobs) {
  const Job &job = jobs.job[blockIdx.y];
  const float *__restrict__ from = job.from;
  for (int64_t e = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4; e < job.all; e += (int64_t)gridDim.x * kThreads * 4) {
    const int n = (int)(job.all - e < 4 ? job.all - e : 4);
    f32x4 s = load4(from + e, n);
    for (int p = 1; p < job.pieces; ++p) s += load4(from + p * job.stride + e, n);
    store4(job.to + e, n, s);
  }
}

// ------------------------------------------------------------------------------ host

constexpr int64_t kMaxTokens = 1 << 24;  // positions that a float of a span holds exactly
constexpr int64_t kMaxGroups = 1 << 24;  // workgroups of a launch: 2^32 lanes

// The head array `a` as [rows, heads, dim]; false where it is none.
bool head_array(const DLArray *a, int heads, int64_t &rows, int64_t &dim) {
  if (a->ndim < 1 || heads < 1) return false;
  const int64_t last = a->shape[a->ndim - 1];
  if (a->ndim == 4) {
    if (a->shape[2] != heads) return false;
    dim = last;
    rows = a->shape[0] * a->shape[1];
  } else {
    if (last % heads != 0) return false;
    dim = last / heads;
    rows = 1;
    for (int i = 0; i + 1 < a->ndim; ++i) rows *= a->shape[i];
  }
  return dim > 0;
}

int describe(const char *what, Call &c, const DLArray *query, const DLArray *key, const DLArray *value, const DLArray *spans,
             const DLArray *slopes, int batch, int heads, int key_heads, float scale, float cap, int causal) {
  auto refuse = [&](const char *why) {
    fprintf(stderr, "[tinyflow_amd] %s: %s\n", what, why);
    return -1;
  };
  if (!on_gpu(query) || !on_gpu(key) || !on_gpu(value)) return refuse("arrays must live on the GPU");
  if (batch < 0 || heads < 1 || key_heads < 1 || heads % key_heads != 0) return refuse("heads must be a multiple of key_heads");
  int64_t q_rows, k_rows, dim, key_dim;
  if (!head_array(query, heads, q_rows, dim) || !head_array(key, key_heads, k_rows, key_dim) || dim != key_dim)
    return refuse("queries and keys must have the same columns a head");
  if (dim > 256) return refuse("heads of more than 256 columns are not supported");
  if (!same_shape(key, value)) return refuse("keys and values must have one shape");
  if (batch == 0 ? q_rows || k_rows : q_rows % batch || k_rows % batch) return refuse("rows must be a multiple of batch");
  const int64_t tq = batch ? q_rows / batch : 0, tk = batch ? k_rows / batch : 0;
  if (tq > kMaxTokens || tk > kMaxTokens) return refuse("more than 2^24 queries or keys of a sequence are not supported");
  if (tq * (heads / key_heads) > INT32_MAX / 2) return refuse("too many queries of a key head");
  if (!(scale > 0.f) || !finite(scale)) return refuse("scale must be positive");
  if (!(cap >= 0.f) || !finite(cap)) return refuse("cap must be positive, or 0 for none");
  // what the kernels make of them (Score): an infinity would turn scores of 0 into NaNs, a number without its digits all of them into others
  if (!finite(cap * kLog2e) || !finite(scale * kLog2e) || (cap > 0.f && !(scale / cap >= 0x1p-126f && finite(scale / cap))))
    return refuse("scale, cap and their quotient must be well inside the range of fp32");
  if (spans) {
    const int64_t n = numel(spans), width = spans->ndim < 2 ? 0 : spans->shape[spans->ndim - 1];
    if (!on_gpu(spans) || (width != 2 && width != 3)) return refuse("spans must be [batch, queries, 2 or 3] or [queries, 2 or 3] and live on the GPU");
    if (n != width * tq && n != width * tq * batch) return refuse("spans must hold two or three numbers for each query");
    c.spans = (const float *)spans->data;
    c.span_width = (int)width;
    c.span_stride = n == width * tq * batch ? width * tq : 0;
  }
  if (slopes) {
    if (!on_gpu(slopes) || numel(slopes) != heads) return refuse("slopes must hold a value for each head and live on the GPU");
    c.slopes = (const float *)slopes->data;
  }
  if (!same_device({query, key, value, spans, slopes})) return refuse("arrays must live on one device");
  c.q = (const float *)query->data;
  c.k = (const float *)key->data;
  c.v = (const float *)value->data;
  c.batch = batch;
  c.tq = (int)tq;
  c.tk = (int)tk;
  c.heads = heads;
  c.key_heads = key_heads;
  c.group = heads / key_heads;
  c.dim = (int)dim;
  c.rows = (int)tq * c.group;
  c.scale = scale;
  c.cap = cap;
  c.causal = causal != 0;
  return 0;
}

template <class F>
void with_columns(int dim, const F &f) {
  if (dim <= 32) f(IC<32>{});
  else if (dim <= 64) f(IC<64>{});
  else if (dim <= 128) f(IC<128>{});
  else f(IC<256>{});
}

// Pieces of a forward tile's walk along the keys: as many as it takes for two workgroups a CU, of 128 keys at least.
int row_pieces(const Call &c, int64_t groups) {
  if (groups == 0) return 1;
  const int64_t wanted = (2 * num_cus() + groups - 1) / groups, most = std::min(kMostPieces, std::max(1, c.tk / 128));
  return (int)std::min<int64_t>(wanted, most);
}

}  // namespace

extern "C" int DLGpuAttentionForward(const DLArrayHandle query, const DLArrayHandle key, const DLArrayHandle value, const DLArrayHandle spans,
                                     const DLArrayHandle slopes, DLArrayHandle output, DLArrayHandle statistics, int batch, int heads,
                                     int key_heads, float scale, float cap, int causal, int *memorytoSaving, void **stream) {
  Call c = {};
  if (describe(__func__, c, query, key, value, spans, slopes, batch, heads, key_heads, scale, cap, causal) != 0) return -1;
  TF_REQUIRE(output || statistics, "no result is asked for");
  TF_REQUIRE(!output || (on_gpu(output) && same_shape(output, query)), "output must live on the GPU and have the query's shape");
  TF_REQUIRE(!statistics || (on_gpu(statistics) && numel(statistics) == (int64_t)batch * heads * c.tq),
             "statistics must hold [batch, heads, queries] values and live on the GPU");
  TF_REQUIRE(same_device({query, output, statistics}), "arrays must live on one device");
  for (const DLArray *read : {(const DLArray *)query, (const DLArray *)key, (const DLArray *)value, (const DLArray *)spans, (const DLArray *)slopes})
    TF_REQUIRE(!overlaps(read, output) && !overlaps(read, statistics), "results must not overlap what they are computed from");
  TF_REQUIRE(!overlaps(output, statistics), "results must not overlap");
  const int64_t all_rows = (int64_t)batch * c.key_heads * c.rows;
  hipStream_t s = stream_of(stream);
  if (all_rows == 0) return 0;
  float *out = output ? (float *)output->data : nullptr, *stat = statistics ? (float *)statistics->data : nullptr;
  const int64_t head_pairs = (int64_t)batch * c.key_heads;
  // (32 rows, 8 heads of 64 over 512 keys, 12 us, by the other forms 21; 5 queries of 4 heads over 4 096 keys, eight sequences, 76 and 177)
  const bool few = c.rows <= 32 && !(c.rows > 16 && c.dim > 128) && (int64_t)c.key_heads * c.dim < 1 << 24;  // 16 rows are less than 2^31 bytes apart
  const bool pairs = !few && pair_suits(c, false);
  int64_t groups;
  int tiles = 0, keys_a_piece = 0;
  Pieces pieces = {};
  pieces.rows = all_rows;
  if (few) {
    // about two workgroups a CU (one each of 2 / 4 / 8: eight sequences of up to 8 192 keys 48 / 53 / 62 us, one of 100 003 51 / 58 / 68); a wave's share of a piece is a multiple of its step
    const int64_t wanted = std::min<int64_t>(kMostPieces, std::max<int64_t>(1, (2 * num_cus() + head_pairs - 1) / head_pairs));
    keys_a_piece = std::max<int>(64, (int)(((c.tk + wanted - 1) / wanted + 63) / 64 * 64));
    pieces.count = std::max(1, (c.tk + keys_a_piece - 1) / keys_a_piece);
    groups = head_pairs * pieces.count;
  } else {
    tiles = (c.rows + kRows - 1) / kRows;
    pieces.count = row_pieces(c, head_pairs * tiles);
    groups = head_pairs * tiles * pieces.count;
  }
  TF_REQUIRE(groups < kMaxGroups, "too many sequences, heads and queries for a launch");
  const size_t planes = pairs ? pair_bytes(c, false) : 0;
  TF_REQUIRE((pieces.count == 1 && !planes) || !being_captured(s), "a pass of this size takes scratch, which a captured stream cannot give back");
  announce_write(output);
  announce_write(statistics);
  char *block = nullptr;
  if (pieces.count > 1 || planes) {
    const size_t marks = pieces.count > 1 ? (size_t)pieces.count * all_rows * sizeof(float2) : 0, sums = marks / sizeof(float2) * c.dim * sizeof(float);
    block = (char *)device_alloc(planes + marks + sums, s);
    if (!block) {
      if (memorytoSaving) *memorytoSaving = shortfall(block_bytes(planes + marks + sums));
      return 0;
    }
    pieces.marks = (float2 *)(block + planes);
    pieces.sums = (float *)(block + planes + marks);
  }
  if (few) {
    auto go = [&](auto dp, auto nc) {
      hipLaunchKernelGGL((few_kernel<decltype(dp)::value, decltype(nc)::value>), dim3((unsigned)groups), dim3(kThreads), 0, s, c, out, stat, pieces, keys_a_piece);
    };
    if (c.rows <= 16) {
      if (c.dim <= 64) go(IC<64>{}, IC<1>{});
      else if (c.dim <= 128) go(IC<128>{}, IC<1>{});
      else go(IC<256>{}, IC<1>{});
    } else {
      if (c.dim <= 64) go(IC<64>{}, IC<2>{});
      else go(IC<128>{}, IC<2>{});
    }
  } else {
    const Exponents left = pairs ? pair_forward(c, out, stat, pieces, tiles, block, s) : Exponents{};
    with_columns(c.dim, [&](auto dp) {
      hipLaunchKernelGGL((rows_kernel<decltype(dp)::value>), dim3((unsigned)groups), dim3(kThreads), 0, s, c, out, stat, pieces, tiles, left);
    });
  }
  if (pieces.count > 1) {
    // one wave a row where the pieces are few: 4 096 keys, eight sequences, 16 pieces, 75 us, with sixteen waves 89
    if (pieces.count > 16) hipLaunchKernelGGL((join_kernel<16>), dim3((unsigned)all_rows), dim3(1024), 0, s, c, pieces, out, stat);
    else hipLaunchKernelGGL((join_kernel<1>), dim3((unsigned)((all_rows + 3) / 4)), dim3(256), 0, s, c, pieces, out, stat);
  }
  if (block) device_free(block, s);
  return finish(s, "DLGpuAttentionForward");
}

extern "C" int DLGpuAttentionBackward(const DLArrayHandle query, const DLArrayHandle key, const DLArrayHandle value, const DLArrayHandle spans,
                                      const DLArrayHandle slopes, const DLArrayHandle output, const DLArrayHandle statistics,
                                      const DLArrayHandle doutput, DLArrayHandle dquery, DLArrayHandle dkey, DLArrayHandle dvalue, int batch,
                                      int heads, int key_heads, float scale, float cap, int causal, int *memorytoSaving, void **stream) {
  Call c = {};
  if (describe(__func__, c, query, key, value, spans, slopes, batch, heads, key_heads, scale, cap, causal) != 0) return -1;
  TF_REQUIRE(on_gpu(output) && on_gpu(doutput) && same_shape(output, query) && same_shape(doutput, query),
             "output and doutput must live on the GPU and have the query's shape");
  TF_REQUIRE(on_gpu(statistics) && numel(statistics) == (int64_t)batch * heads * c.tq, "statistics must hold [batch, heads, queries] values and live on the GPU");
  TF_REQUIRE(dquery || dkey || dvalue, "no gradient is asked for");
  TF_REQUIRE(!dquery || (on_gpu(dquery) && same_shape(dquery, query)), "dquery must live on the GPU and have the query's shape");
  TF_REQUIRE(!dkey || (on_gpu(dkey) && same_shape(dkey, key)), "dkey must live on the GPU and have the key's shape");
  TF_REQUIRE(!dvalue || (on_gpu(dvalue) && same_shape(dvalue, value)), "dvalue must live on the GPU and have the value's shape");
  TF_REQUIRE(same_device({query, output, statistics, doutput, dquery, dkey, dvalue}), "arrays must live on one device");
  for (const DLArray *read : {(const DLArray *)query, (const DLArray *)key, (const DLArray *)value, (const DLArray *)spans, (const DLArray *)slopes,
                              (const DLArray *)output, (const DLArray *)statistics, (const DLArray *)doutput})
    for (const DLArray *written : {(const DLArray *)dquery, (const DLArray *)dkey, (const DLArray *)dvalue})
      TF_REQUIRE(!overlaps(read, written), "gradients must not overlap what they are computed from");
  TF_REQUIRE(!overlaps(dquery, dkey) && !overlaps(dquery, dvalue) && !overlaps(dkey, dvalue), "gradients must not overlap");
  hipStream_t s = stream_of(stream);
  const int64_t head_pairs = (int64_t)batch * c.key_heads, all_rows = head_pairs * c.rows, all_keys = head_pairs * c.tk;
  if (all_rows == 0 && all_keys == 0) return 0;
  const int row_tiles = (c.rows + kRows - 1) / kRows, key_tiles = (c.tk + kRows - 1) / kRows;
  const int64_t key_groups = head_pairs * key_tiles;
  const bool pairs = all_rows && all_keys && pair_suits(c, true);
  // Where the tiles leave CUs without work their walks are cut, in pieces of 128 or more rows or keys (of 256: one head of 64, backward, 256 x 256 47.5 us and
  // here 44.5, 300 x 1000 60 and 49).  Cutting dq as well took 8 queries over 8 192 keys from 320 us to 55, and from 1 288 to 59 on the fp32 instruction.
  // Two workgroups a CU: with four, two of which fit one with short heads, 4 x 1 024 tokens of 16 heads of 64 took 200 us, with two 177.
  int pieces = 1, row_pieces = 1;
  const int64_t row_groups = head_pairs * row_tiles;
  if ((dkey || dvalue) && key_groups) pieces = (int)std::min<int64_t>((2 * num_cus() + key_groups - 1) / key_groups, std::max(1, c.rows / 128));
  if (dquery && row_groups) row_pieces = (int)std::min<int64_t>((2 * num_cus() + row_groups - 1) / row_groups, std::max(1, c.tk / 128));
  TF_REQUIRE(row_groups * row_pieces < kMaxGroups && key_groups * pieces < kMaxGroups && (all_rows + 3) / 4 < kMaxGroups,
             "too many sequences, heads and queries for a launch");
  TF_REQUIRE(!being_captured(s), "the backward pass takes scratch, which a captured stream cannot give back");
  for (const DLArray *written : {(const DLArray *)dquery, (const DLArray *)dkey, (const DLArray *)dvalue}) announce_write(written);
  const int64_t all = all_keys * c.dim, all_queries = all_rows * c.dim;
  const size_t row_bytes = (size_t)all_rows * sizeof(Row), row_part_bytes = row_pieces > 1 ? (size_t)row_pieces * all_queries * sizeof(float) : 0;
  const size_t part_bytes = pieces > 1 ? (size_t)pieces * 2 * all * sizeof(float) : 0;
  const size_t planes = pairs ? pair_bytes(c, true) : 0, bytes = planes + row_bytes + row_part_bytes + part_bytes;
  char *block = (char *)device_alloc(bytes, s);
  if (!block) {
    if (memorytoSaving) *memorytoSaving = shortfall(block_bytes(bytes));
    return 0;
  }
  Row *rows = (Row *)(block + planes);
  float *row_parts = (float *)(block + planes + row_bytes), *parts = (float *)(block + planes + row_bytes + row_part_bytes);
  const float *dout = (const float *)doutput->data;
  float *dq = dquery ? (float *)dquery->data : nullptr, *dk = dkey ? (float *)dkey->data : nullptr, *dv = dvalue ? (float *)dvalue->data : nullptr;
  const Gradients to = {row_pieces > 1 ? row_parts : dq, dk, dv, parts, row_pieces > 1 ? all_queries : 0, row_pieces, pieces};
  if (all_rows && !pairs)
    hipLaunchKernelGGL(prepare_kernel, dim3((unsigned)((all_rows + 3) / 4)), dim3(kThreads), 0, s, c, (const float *)output->data,
                       (const float *)statistics->data, dout, rows, all_rows);
  const Exponents left =
      pairs ? pair_backward(c, (const float *)output->data, (const float *)statistics->data, dout, rows, to, row_tiles, key_tiles, block, s) : Exponents{};
  with_columns(c.dim, [&](auto columns) {
    constexpr int DP = decltype(columns)::value;
    if (dq && all_rows)
      hipLaunchKernelGGL((dq_kernel<DP>), dim3((unsigned)(row_groups * row_pieces)), dim3(kThreads), 0, s, c, dout, rows, to.dq, to.row_stride, row_tiles, row_pieces, left);
    if (!key_groups) return;
    const dim3 grid((unsigned)(key_groups * pieces));
    if constexpr (DP <= 128) {
      if (dk && dv) {
        hipLaunchKernelGGL((dkv_kernel<DP, true, true>), grid, dim3(kThreads), 0, s, c, dout, rows, dk, dv, parts, key_tiles, pieces, left);
        return;
      }
    }
    // heads of more than 128 columns: the operands and sums of one gradient fill the registers
    if (dk) hipLaunchKernelGGL((dkv_kernel<DP, true, false>), grid, dim3(kThreads), 0, s, c, dout, rows, dk, nullptr, parts, key_tiles, pieces, left);
    if (dv) hipLaunchKernelGGL((dkv_kernel<DP, false, true>), grid, dim3(kThreads), 0, s, c, dout, rows, nullptr, dv, parts, key_tiles, pieces, left);
  });
  Jobs sums = {};
  if (row_pieces > 1) sums.job[sums.n++] = Job{row_parts, dq, all_queries, all_queries, row_pieces};
  if (pieces > 1 && dk) sums.job[sums.n++] = Job{parts, dk, all, 2 * all, pieces};
  if (pieces > 1 && dv) sums.job[sums.n++] = Job{parts + all, dv, all, 2 * all, pieces};
  if (sums.n) {
    const int64_t most = std::max(row_pieces > 1 ? all_queries : 0, pieces > 1 ? all : 0);
    hipLaunchKernelGGL(sum_kernel, dim3((unsigned)std::min<int64_t>((most / 4 + kThreads) / kThreads, 4 * num_cus()), sums.n), dim3(kThreads), 0, s, sums);
  }
  device_free(block, s);
  return finish(s, "DLGpuAttentionBackward");
}
