// What the heads of queries, keys and values go through between their projection and attention: the norm of each head's
// vector, the rotation of its columns by position, and the row of a cache that they are written to (no counterpart in the reference).
//
//   s = 1 / sqrt(mean(x^2) + eps), n = x s, y = n gamma                       over a head's columns; without gamma y = x
//   (a, b) -> amplitude (a cos t - b sin t, a sin t + b cos t), t = position frequency   for pairs of the first `rotary` columns
//   backward: da is dy rotated by -t, c = mean(da gamma n), dx = s (da gamma - n c), dgamma = sum over rows and heads of da n
//
// Nothing is kept between the two passes: x is in registers anyway, and the angles cost less than reading them.
//
// Bound: HBM.  A lane holds eight columns, four and the four that they are paired with (the four behind them where pairs are neighbours),
// so no pair is split between lanes; 8 to 64 lanes hold a head's vector.  All heads of a row have its angles: a group of lanes
// computes them once for the heads that it takes one after the other.  Angles are products and remainders in 64 bits (a
// position past 2^20 times a frequency near 1 has no digits left behind the point in 32); what is left, at most an eighth of a turn, goes to sine
// and cosine in 32.
#include "internal.h"
#include "lanes.h"

#include <algorithm>

using namespace tf;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));  // rows of any length start anywhere: 16-byte accesses on 4-byte alignment

constexpr int kThreads = 256;
constexpr int kMaxParts = 4, kMaxDim = 1024;
constexpr int kMaxGroups = 1 << 24;  // workgroups of a launch: 2^32 lanes

struct Part {
  const float *x, *gamma, *dy;
  float *out;       // y or dx
  float *partial;   // [workgroup of the part][dim], the weights' gradients; null: not asked for
  int heads, chunks;  // chunks: groups of heads that share a row's angles
  bool rotate, place;
  int first_group, groups;
};

struct Launch {
  Part parts[kMaxParts];
  int n_parts;
  const float *positions, *frequencies, *slots;
  int64_t rows, n_positions, row_slots, capacity;  // row_slots: rows of a sequence, with slots
  int dim, rotary, heads_a_chunk;
  bool interleaved;
  float amplitude, eps, n;
};

// The columns of a lane's unit: `a` and the up to four behind it, `b` likewise.
template <bool WHOLE>
struct Unit {
  int a, b, count_a, count_b, pair;  // pair < 0: not rotated
  __device__ inline Unit(int u, int dim, int rotary, bool interleaved) {
    const int half = rotary / 2, rotated = interleaved ? (rotary + 7) / 8 : (half + 3) / 4;
    if (u < rotated) {
      pair = 4 * u;
      a = interleaved ? 8 * u : 4 * u;
      b = interleaved ? 8 * u + 4 : half + 4 * u;
      count_a = interleaved ? min(4, rotary - a) : min(4, half - a);
      count_b = interleaved ? max(0, min(4, rotary - b)) : count_a;
    } else {
      pair = -1;
      a = rotary + 8 * (u - rotated);
      b = a + 4;
      count_a = max(0, min(4, dim - a));
      count_b = max(0, min(4, dim - b));
    }
    if (WHOLE) count_a = count_b = 4;
  }
};

__device__ inline f32x4 load(const float *p, int count) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (count == 4) return *reinterpret_cast<const f32x4u *>(p);
  if (count > 0) v[0] = p[0];
  if (count > 1) v[1] = p[1];
  if (count > 2) v[2] = p[2];
  return v;
}
__device__ inline void store(float *p, int count, f32x4 v) {
  if (count == 4) *reinterpret_cast<f32x4u *>(p) = v;
  else {
    if (count > 0) p[0] = v[0];
    if (count > 1) p[1] = v[1];
    if (count > 2) p[2] = v[2];
  }
}

// A row's cosines and sines, times the amplitude, of a unit's four pairs.
struct Turn {
  f32x4 c, s;
  __device__ inline void set(const Launch &l, float position, f32x4 frequency) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = frequency[e];
      const double quarters = (double)position * (double)f * 0.63661977236758134308;  // 2 / pi
      const double whole = rint(quarters);
      float sine, cosine;
      sincospif((float)(quarters - whole) * 0.5f, &sine, &cosine);
      // the whole quarters modulo four, also of numbers that no integer holds; an infinity or a NaN has left a NaN
      const int q = (int)(whole - 4.0 * floor(whole * 0.25));
      const float cs = q & 1 ? -sine : cosine, sn = q & 1 ? cosine : sine;
      c[e] = (q & 2 ? -cs : cs) * l.amplitude;
      s[e] = (q & 2 ? -sn : sn) * l.amplitude;
    }
  }
};

// backward: by the opposite angle
template <bool BACKWARD>
__device__ inline void rotate(f32x4 &a, f32x4 &b, const Turn &t, bool interleaved) {
  const f32x4 s = BACKWARD ? -t.s : t.s;
  if (interleaved) {
    const f32x4 x = a, y = b;
    a = f32x4{x[0] * t.c[0] - x[1] * s[0], x[0] * s[0] + x[1] * t.c[0], x[2] * t.c[1] - x[3] * s[1], x[2] * s[1] + x[3] * t.c[1]};
    b = f32x4{y[0] * t.c[2] - y[1] * s[2], y[0] * s[2] + y[1] * t.c[2], y[2] * t.c[3] - y[3] * s[3], y[2] * s[3] + y[3] * t.c[3]};
  } else {
    const f32x4 x = a;
    a = x * t.c - b * s;
    b = x * s + b * t.c;
  }
}

__device__ inline float dot(f32x4 a, f32x4 b) { return (a[0] * b[0] + a[1] * b[1]) + (a[2] * b[2] + a[3] * b[3]); }

__device__ inline int part_of(const Launch &l, int group) {
  int p = 0;
  for (int i = 1; i < l.n_parts; ++i) p = group >= l.parts[i].first_group ? i : p;
  return p;
}

// Where row r of a part is written, or -1.
__device__ inline int64_t row_out(const Launch &l, const Part &part, int64_t r) {
  if (!part.place) return r;
  const float slot = l.slots[r];
  if (!(slot >= 0.f && slot < (float)l.capacity && slot == floorf(slot))) return -1;
  return r / l.row_slots * l.capacity + (int64_t)slot;
}

// The frequencies of a unit's four pairs.
template <bool WHOLE>
__device__ inline f32x4 frequencies_of(const Launch &l, const Unit<WHOLE> &unit) {
  if (unit.pair < 0) return f32x4{0.f, 0.f, 0.f, 0.f};
  return load(l.frequencies + unit.pair, WHOLE ? 4 : min(4, l.rotary / 2 - unit.pair));
}

// T lanes a head, U units a lane; WHOLE: every lane's units are whole, so that no load stands behind a branch.  A head is loaded before what the one in front of it
// needs is computed, the first before the angles.  (4 096 rows of 16 + 4 heads of 128 17.0 us without and 14.2, 5.9 TB/s; backward 27.3 and 26.1.)
template <int T, int U, bool WHOLE>
__global__ __launch_bounds__(kThreads) void forward_kernel(const Launch l) {
  const int p = part_of(l, (int)blockIdx.x);
  const Part &part = l.parts[p];
  const int lane = threadIdx.x % T;
  const int64_t item = ((int64_t)blockIdx.x - part.first_group) * (kThreads / T) + threadIdx.x / T;
  const int64_t r = item / part.chunks;
  if (r >= l.rows) return;  // lanes of a head together
  const int chunk = (int)(item % part.chunks), first = chunk * l.heads_a_chunk, end = min(part.heads, first + l.heads_a_chunk);
  const int rotary = part.rotate ? l.rotary : 0;
  const float *x = part.x + (r * part.heads + first) * l.dim;
  const float position = part.rotate ? l.positions[r % l.n_positions] : 0.f;
  f32x4 ga[U], gb[U], next_a[U], next_b[U], frequency[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
    next_a[u] = load(x + unit.a, unit.count_a);
    next_b[u] = load(x + unit.b, unit.count_b);
    frequency[u] = frequencies_of(l, unit);
    if (part.gamma) {
      ga[u] = load(part.gamma + unit.a, unit.count_a);
      gb[u] = load(part.gamma + unit.b, unit.count_b);
    }
  }
  const int64_t to = row_out(l, part, r);
  if (to < 0) return;
  Turn turn[U];
  if (part.rotate)
#pragma unroll
    for (int u = 0; u < U; ++u) turn[u].set(l, position, frequency[u]);
  float *y = part.out + (to * part.heads + first) * l.dim;
  for (int h = first; h < end; ++h, y += l.dim) {
    f32x4 a[U], b[U];
    float squares = 0.f;
    x += h + 1 < end ? l.dim : 0;  // the last one again
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
      a[u] = next_a[u];
      b[u] = next_b[u];
      next_a[u] = load(x + unit.a, unit.count_a);
      next_b[u] = load(x + unit.b, unit.count_b);
      squares += dot(a[u], a[u]) + dot(b[u], b[u]);
    }
    if (part.gamma) {
      const float s = 1.f / sqrtf(lanes::sum_over<T>(squares) / l.n + l.eps);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u] = a[u] * s * ga[u];
        b[u] = b[u] * s * gb[u];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
      if (unit.pair >= 0) rotate<false>(a[u], b[u], turn[u], l.interleaved);
      store(y + unit.a, unit.count_a, a[u]);
      store(y + unit.b, unit.count_b, b[u]);
    }
  }
}

// A part's workgroups take its items in turn; each lane keeps the sums of da n of its columns.
template <int T, int U, bool WHOLE>
__global__ __launch_bounds__(kThreads) void backward_kernel(const Launch l) {
  const int p = part_of(l, (int)blockIdx.x);
  const Part &part = l.parts[p];
  constexpr int GROUPS = kThreads / T;
  const int lane = threadIdx.x % T, sub = threadIdx.x / T;
  const int rotary = part.rotate ? l.rotary : 0;
  f32x4 ga[U], gb[U], sum_a[U], sum_b[U], frequency[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
    frequency[u] = frequencies_of(l, unit);
    if (part.gamma) {
      ga[u] = load(part.gamma + unit.a, unit.count_a);
      gb[u] = load(part.gamma + unit.b, unit.count_b);
    }
    sum_a[u] = sum_b[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int64_t items = l.rows * part.chunks;
  const int group = (int)blockIdx.x - part.first_group;
  for (int64_t item = (int64_t)group * GROUPS + sub; item < items; item += (int64_t)part.groups * GROUPS) {
    const int64_t r = item / part.chunks;
    const int first = (int)(item % part.chunks) * l.heads_a_chunk, end = min(part.heads, first + l.heads_a_chunk);
    const float position = part.rotate ? l.positions[r % l.n_positions] : 0.f;
    const int64_t at = (r * part.heads + first) * l.dim;
    const float *x = part.x + at, *dy = part.dy + at;
    float *dx = part.out ? part.out + at : nullptr;
    f32x4 next_a[U], next_b[U], next_da[U], next_db[U];
    auto fetch = [&]() {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
        next_da[u] = load(dy + unit.a, unit.count_a);
        next_db[u] = load(dy + unit.b, unit.count_b);
        if (part.gamma) {
          next_a[u] = load(x + unit.a, unit.count_a);
          next_b[u] = load(x + unit.b, unit.count_b);
        }
      }
    };
    fetch();
    Turn turn[U];
    if (part.rotate)
#pragma unroll
      for (int u = 0; u < U; ++u) turn[u].set(l, position, frequency[u]);
    for (int h = first; h < end; ++h, dx += dx ? l.dim : 0) {
      f32x4 a[U], b[U], da[U], db[U];
      float squares = 0.f, products = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        da[u] = next_da[u];
        db[u] = next_db[u];
        if (part.gamma) {
          a[u] = next_a[u];
          b[u] = next_b[u];
        }
      }
      const int step = h + 1 < end ? l.dim : 0;  // the last one again
      x += step;
      dy += step;
      fetch();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
        if (part.gamma) squares += dot(a[u], a[u]) + dot(b[u], b[u]);
        if (unit.pair >= 0) rotate<true>(da[u], db[u], turn[u], l.interleaved);
      }
      if (part.gamma) {
        const float s = 1.f / sqrtf(lanes::sum_over<T>(squares) / l.n + l.eps);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          a[u] *= s;
          b[u] *= s;
          sum_a[u] += da[u] * a[u];
          sum_b[u] += db[u] * b[u];
          da[u] *= ga[u];
          db[u] *= gb[u];
          products += dot(da[u], a[u]) + dot(db[u], b[u]);
        }
        const float c = lanes::sum_over<T>(products) / l.n;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          da[u] = (da[u] - a[u] * c) * s;
          db[u] = (db[u] - b[u] * c) * s;
        }
      }
      if (dx) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
          store(dx + unit.a, unit.count_a, da[u]);
          store(dx + unit.b, unit.count_b, db[u]);
        }
      }
    }
  }
  if (!part.partial) return;  // of the whole workgroup
  __shared__ f32x4 sums[GROUPS][2 * U][T];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    sums[sub][2 * u][lane] = sum_a[u];
    sums[sub][2 * u + 1][lane] = sum_b[u];
  }
  __syncthreads();
  if (sub > 0) return;
  float *to = part.partial + (int64_t)group * l.dim;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Unit<WHOLE> unit(u * T + lane, l.dim, rotary, l.interleaved);
    for (int g = 1; g < GROUPS; ++g) {
      sum_a[u] += sums[g][2 * u][lane];
      sum_b[u] += sums[g][2 * u + 1][lane];
    }
    store(to + unit.a, unit.count_a, sum_a[u]);
    store(to + unit.b, unit.count_b, sum_b[u]);
  }
}

struct Sums {
  const float *partial[kMaxParts];
  float *dgamma[kMaxParts];
  int pieces[kMaxParts];
};

// dgamma of the part blockIdx.y: 32 columns a workgroup, every 32nd partial sum a lane, added up in their order.  No pieces: zeros.
__global__ __launch_bounds__(1024) void sum_pieces_kernel(const Sums of, int dim) {
  __shared__ float sums[32][33];
  const int along = threadIdx.x % 32, slice = threadIdx.x / 32, c = blockIdx.x * 32 + along;
  const float *partial = of.partial[blockIdx.y];
  float s = 0.f;
  const int pieces = of.pieces[blockIdx.y];
  if (c < dim)
    for (int p = slice; p < pieces; p += 32 * 8) {  // eight loads under way
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = partial[(int64_t)min(p + 32 * e, pieces - 1) * dim + c];
#pragma unroll
      for (int e = 0; e < 8; ++e) s += p + 32 * e < pieces ? v[e] : 0.f;
    }
  sums[slice][along] = s;
  __syncthreads();
  if (slice > 0 || c >= dim) return;
  for (int w = 1; w < 32; ++w) s += sums[w][along];
  of.dgamma[blockIdx.y][c] = s;
}

// The columns of a head of an array: axes 2 and 3 of a rank of four, the last axis in `heads` parts of any other.  0: neither.
int64_t head_dim(const DLArray *a, int heads) {
  if (a->ndim < 1 || heads < 1) return 0;
  const int64_t last = a->shape[a->ndim - 1];
  if (a->ndim == 4) return a->shape[2] == heads ? last : 0;
  return last % heads == 0 ? last / heads : 0;
}

// What both directions check and set for all parts; `what` names the call in messages.
int common(const char *what, Launch &l, const DLArray *positions, const DLArray *frequencies, int64_t rows, int64_t dim, bool rotates,
           float amplitude, int interleaved, float eps, const DLArray *first) {
  auto refuse = [&](const char *why) {
    fprintf(stderr, "[tinyflow_amd] %s: %s\n", what, why);
    return -1;
  };
  if (dim < 1 || dim > kMaxDim) return refuse("heads must have 1 to 1024 columns");
  if (!(eps >= 0.f)) return refuse("eps must not be negative");
  l.rows = rows;
  l.dim = (int)dim;
  l.n = (float)dim;
  l.amplitude = amplitude;
  l.interleaved = interleaved != 0;
  l.eps = eps;
  if (!rotates) return 0;
  if (!on_gpu(positions) || !on_gpu(frequencies)) return refuse("positions and frequencies must live on the GPU");
  if (!same_device({first, positions, frequencies})) return refuse("arrays must live on one device");
  l.n_positions = numel(positions);
  l.rotary = (int)std::min<int64_t>(2 * numel(frequencies), dim + 1);
  if (frequencies->ndim != 1 || l.rotary > dim) return refuse("frequencies must hold one value for each pair of columns, half of a head's at most");
  if (rows && (l.n_positions == 0 || rows % l.n_positions != 0)) return refuse("positions must hold one value for each row, or for each of a sequence that the rows repeat");
  l.positions = (const float *)positions->data;
  l.frequencies = (const float *)frequencies->data;
  return 0;
}

// Lanes a head and units a lane.
template <class F>
void with_lanes(const Launch &l, const F &f) {
  // the unrotated part of a head may leave one unit more than its columns fill
  const int rotated = l.interleaved ? (l.rotary + 7) / 8 : (l.rotary / 2 + 3) / 4;
  const int units = std::max(rotated + (l.dim - l.rotary + 7) / 8, (l.dim + 7) / 8);
  auto go = [&](auto t, auto u) {
    // all lanes' units are whole
    if (l.dim == 8 * decltype(t)::value * decltype(u)::value && l.rotary % 8 == 0) f(t, u, std::true_type{});
    else f(t, u, std::false_type{});
  };
  if (units <= 8) go(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
  else if (units <= 16) go(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  else if (units <= 32) go(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  else if (units <= 64) go(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  else f(std::integral_constant<int, 64>{}, std::integral_constant<int, 3>{}, std::false_type{});  // up to 1 024 of 1 536 columns
}

// Heads that share a row's angles: one where lanes are few, up to four where there are enough of them.  Microseconds with one, two and four, forward /
// backward: 256 rows of 16 + 4 heads of 128 5.9 / 9.1, 6.1 / 11.1, 6.9 / 11.0; 1 024 rows 8.2 / 15.5, 7.8 / 12.4, 8.3 / 12.8; 4 096 rows 21.3 / 33.8,
// 17.4 / 30.1, 17.1 / 30.2; 4 096 rows of 64 12.0 / 25.0, 10.4 / 22.4, 10.4 / 18.2; eight are slower everywhere.
void set_chunks(Launch &l, int64_t total_heads) {
  const int64_t heads = l.rows * total_heads;
  l.heads_a_chunk = heads >= 65536 ? 4 : heads >= 16384 ? 2 : 1;
  for (int i = 0; i < l.n_parts; ++i) l.parts[i].chunks = (l.parts[i].heads + l.heads_a_chunk - 1) / l.heads_a_chunk;
}

}  // namespace

extern "C" int DLGpuHeadRotary(const DLHeadPart *parts, int n_parts, const DLArrayHandle positions, const DLArrayHandle frequencies,
                               float amplitude, int interleaved, float eps, const DLArrayHandle slots, void **stream) {
  TF_REQUIRE(parts && n_parts >= 1 && n_parts <= kMaxParts, "one to four parts are supported");
  Launch l = {};
  l.n_parts = n_parts;
  bool rotates = false, places = false;
  int64_t rows = 0, dim = 0, total_heads = 0;
  for (int i = 0; i < n_parts; ++i) {
    const DLHeadPart &p = parts[i];
    TF_REQUIRE(on_gpu(p.input) && on_gpu(p.output), "arrays must live on the GPU");
    const int64_t d = head_dim(p.input, p.heads);
    TF_REQUIRE(d > 0 && d <= kMaxDim, "an input's columns must be those of its heads, 1 to 1024 each");
    const int64_t n = numel(p.input) / (d * p.heads);
    if (i == 0) rows = n, dim = d;
    TF_REQUIRE(n == rows && d == dim, "the parts must have the same rows and columns a head");
    if (p.place) {
      TF_REQUIRE(head_dim(p.output, p.heads) == d, "an output's columns must be those of its heads");
    } else {
      TF_REQUIRE(same_shape(p.input, p.output), "an output must have its input's shape");
    }
    if (p.gamma) TF_REQUIRE(on_gpu(p.gamma) && p.gamma->ndim == 1 && p.gamma->shape[0] == d, "gamma must hold one value for each column of a head");
    TF_REQUIRE(same_device({parts[0].input, p.input, p.output, p.gamma}), "arrays must live on one device");
    rotates |= p.rotate != 0;
    places |= p.place != 0;
    total_heads += p.heads;
    l.parts[i] = Part{(const float *)p.input->data, p.gamma ? (const float *)p.gamma->data : nullptr, nullptr, (float *)p.output->data,
                      nullptr, p.heads, 0, p.rotate != 0, p.place != 0, 0, 0};
  }
  if (common(__func__, l, positions, frequencies, rows, dim, rotates, amplitude, interleaved, eps, parts[0].input) != 0) return -1;
  if (places) {
    TF_REQUIRE(on_gpu(slots) && slots->ndim == 2 && numel(slots) == rows, "slots must be [sequences, rows of a sequence] and live on the GPU");
    TF_REQUIRE(same_device({parts[0].input, slots}), "arrays must live on one device");
    l.slots = (const float *)slots->data;
    l.row_slots = slots->shape[1];
    const int64_t sequences = slots->shape[0];
    bool first = true;
    for (int i = 0; i < n_parts; ++i) {
      if (!parts[i].place) continue;
      const int64_t out_rows = numel(parts[i].output) / (dim * parts[i].heads);
      TF_REQUIRE(sequences == 0 ? out_rows == 0 : out_rows % sequences == 0, "a placed output must hold the same rows for each sequence");
      const int64_t capacity = sequences ? out_rows / sequences : 0;
      TF_REQUIRE(first || capacity == l.capacity, "placed outputs must hold the same rows for each sequence");
      TF_REQUIRE(capacity <= 1 << 24, "slots count up to 2^24 rows");
      l.capacity = capacity;
      first = false;
    }
  }
  for (int i = 0; i < n_parts; ++i) {
    const DLArray *out = parts[i].output;
    for (int j = 0; j < n_parts; ++j) {
      TF_REQUIRE(i == j || !overlaps(out, parts[j].output), "outputs must not overlap");
      TF_REQUIRE(!overlaps(out, parts[j].gamma), "outputs must not overlap gammas");
      TF_REQUIRE((i == j && !parts[i].place && out->data == parts[j].input->data) || !overlaps(out, parts[j].input),
                 "an output must be its own input or overlap none");
    }
    if (rotates) TF_REQUIRE(!overlaps(out, positions) && !overlaps(out, frequencies), "outputs must not overlap positions or frequencies");
    if (places) TF_REQUIRE(!overlaps(out, slots), "outputs must not overlap slots");
  }
  set_chunks(l, total_heads);
  int64_t groups = 0;
  with_lanes(l, [&](auto t, auto, auto) {
    for (int i = 0; i < n_parts; ++i) {
      const int64_t a_group = kThreads / decltype(t)::value;
      l.parts[i].first_group = (int)std::min<int64_t>(groups, kMaxGroups);
      groups += (l.rows * l.parts[i].chunks + a_group - 1) / a_group;
    }
  });
  TF_REQUIRE(groups < kMaxGroups, "too many rows and heads for a launch");
  for (int i = 0; i < n_parts; ++i) announce_write(parts[i].output);
  hipStream_t s = stream_of(stream);
  if (groups == 0) return 0;
  with_lanes(l, [&](auto t, auto u, auto whole) {
    hipLaunchKernelGGL((forward_kernel<decltype(t)::value, decltype(u)::value, decltype(whole)::value>), dim3((unsigned)groups), dim3(kThreads), 0, s, l);
  });
  return finish(s, "DLGpuHeadRotary");
}

extern "C" int DLGpuHeadRotaryBackward(const DLHeadGradientPart *parts, int n_parts, const DLArrayHandle positions,
                                       const DLArrayHandle frequencies, float amplitude, int interleaved, float eps,
                                       int *memorytoSaving, void **stream) {
  TF_REQUIRE(parts && n_parts >= 1 && n_parts <= kMaxParts, "one to four parts are supported");
  Launch l = {};
  l.n_parts = n_parts;
  bool rotates = false, sums = false;
  int64_t rows = 0, dim = 0, total_heads = 0;
  for (int i = 0; i < n_parts; ++i) {
    const DLHeadGradientPart &p = parts[i];
    TF_REQUIRE(on_gpu(p.doutput), "arrays must live on the GPU");
    const int64_t d = head_dim(p.doutput, p.heads);
    TF_REQUIRE(d > 0 && d <= kMaxDim, "a gradient's columns must be those of its heads, 1 to 1024 each");
    const int64_t n = numel(p.doutput) / (d * p.heads);
    if (i == 0) rows = n, dim = d;
    TF_REQUIRE(n == rows && d == dim, "the parts must have the same rows and columns a head");
    TF_REQUIRE(p.dinput || p.dgamma, "a part without a gradient to compute");
    if (p.dinput) TF_REQUIRE(on_gpu(p.dinput) && same_shape(p.dinput, p.doutput), "dinput must live on the GPU and have doutput's shape");
    if (p.gamma) {
      TF_REQUIRE(on_gpu(p.gamma) && p.gamma->ndim == 1 && p.gamma->shape[0] == d, "gamma must hold one value for each column of a head");
      TF_REQUIRE(on_gpu(p.input) && same_shape(p.input, p.doutput), "a normed input must live on the GPU and have doutput's shape");
    }
    if (p.dgamma) TF_REQUIRE(p.gamma && on_gpu(p.dgamma) && same_shape(p.gamma, p.dgamma), "dgamma must live on the GPU and have gamma's shape");
    TF_REQUIRE(same_device({parts[0].doutput, p.doutput, p.dinput, p.gamma, p.gamma ? p.input : nullptr, p.dgamma}), "arrays must live on one device");
    rotates |= p.rotate != 0;
    sums |= p.dgamma != nullptr;
    total_heads += p.heads;
    l.parts[i] = Part{p.gamma ? (const float *)p.input->data : nullptr, p.gamma ? (const float *)p.gamma->data : nullptr,
                      (const float *)p.doutput->data, p.dinput ? (float *)p.dinput->data : nullptr, nullptr, p.heads, 0, p.rotate != 0, false, 0, 0};
  }
  if (common(__func__, l, positions, frequencies, rows, dim, rotates, amplitude, interleaved, eps, parts[0].doutput) != 0) return -1;
  for (int i = 0; i < n_parts; ++i)
    for (const DLArray *written : {(const DLArray *)parts[i].dinput, (const DLArray *)parts[i].dgamma}) {
      for (int j = 0; j < n_parts; ++j) {
        TF_REQUIRE(!overlaps(written, parts[j].gamma ? parts[j].input : nullptr) && !overlaps(written, parts[j].gamma),
                   "gradients must not overlap what they are computed from");
        TF_REQUIRE((i == j && written == parts[i].dinput && written && written->data == parts[j].doutput->data) || !overlaps(written, parts[j].doutput),
                   "a gradient must be its own doutput or overlap none");
        for (const DLArray *other : {(const DLArray *)parts[j].dinput, (const DLArray *)parts[j].dgamma})
          TF_REQUIRE(other == written || !overlaps(written, other), "gradients must not overlap");
        TF_REQUIRE(i == j || !written || (written != parts[j].dinput && written != parts[j].dgamma), "gradients must not overlap");
      }
      if (rotates) TF_REQUIRE(!overlaps(written, positions) && !overlaps(written, frequencies), "gradients must not overlap what they are computed from");
    }
  for (int i = 0; i < n_parts; ++i) {
    announce_write(parts[i].dinput);
    announce_write(parts[i].dgamma);
  }
  hipStream_t s = stream_of(stream);
  TF_REQUIRE(!sums || !being_captured(s), "the gradients of the weights take scratch, which a captured stream cannot give back");
  set_chunks(l, total_heads);
  // A part's workgroups: up to eight a CU for all parts, in the proportion of their heads, each with a partial sum of the weights' gradients.  (4 096 rows
  // of 16 + 4 heads of 128: 27.3 us; up to four 30.3, one 41.7.)
  int64_t groups = 0, pieces = 0;
  with_lanes(l, [&](auto t, auto, auto) {
    for (int i = 0; i < n_parts; ++i) {
      const int64_t a_group = kThreads / decltype(t)::value, wanted = (l.rows * l.parts[i].chunks + a_group - 1) / a_group;
      const int64_t most = std::max<int64_t>(1, (int64_t)8 * num_cus() * l.parts[i].heads / total_heads);
      l.parts[i].first_group = (int)groups;
      l.parts[i].groups = (int)std::min(wanted, most);
      groups += l.parts[i].groups;
      if (parts[i].dgamma) pieces += l.parts[i].groups;
    }
  });
  float *partial = nullptr;
  if (pieces) {
    const size_t bytes = (size_t)pieces * dim * sizeof(float);
    partial = (float *)device_alloc(bytes, s);
    if (!partial) {
      if (memorytoSaving) *memorytoSaving = shortfall(block_bytes(bytes));
      return 0;
    }
  }
  Sums of = {};
  int n_sums = 0;
  float *at = partial;
  for (int i = 0; i < n_parts; ++i) {
    if (!parts[i].dgamma) continue;
    l.parts[i].partial = at;
    of.partial[n_sums] = at;
    of.dgamma[n_sums] = (float *)parts[i].dgamma->data;
    of.pieces[n_sums++] = l.parts[i].groups;
    at += (int64_t)l.parts[i].groups * dim;
  }
  if (groups)
    with_lanes(l, [&](auto t, auto u, auto whole) {
      hipLaunchKernelGGL((backward_kernel<decltype(t)::value, decltype(u)::value, decltype(whole)::value>), dim3((unsigned)groups), dim3(kThreads), 0, s, l);
    });
  if (n_sums) hipLaunchKernelGGL(sum_pieces_kernel, dim3((unsigned)((dim + 31) / 32), (unsigned)n_sums), dim3(1024), 0, s, of, (int)dim);
  if (partial) device_free(partial, s);
  return finish(s, "DLGpuHeadRotaryBackward");
}
