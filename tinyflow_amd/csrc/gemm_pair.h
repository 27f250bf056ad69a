// Large fp32 products on the fp16 matrix instruction, from operands that a pass before has split.
//
//   D[m, n] = sum_k A(m, k) B(n, k)
//
// Every row of A and of B (all that enters one sum) is multiplied by the power of two that brings its largest value into
// [2^14, 2^15), and each element is then made of two fp16 numbers, x = h + 2^-11 l: h its nearest one, l the nearest of 2^11 times what
// is left.  h keeps 11 significant bits, and l eleven of the remaining thirteen and a sign, so at most 2^-23 of x is left off, as
// long as neither leaves the normal numbers: for everything down to 2^-27 of its row's largest value.  Below that the error stays at
// 2^-36, which is 2^-50 of that value at most, where an fp32 product of rows of unlike magnitudes would go on being exact.  (Without the factor
// 2^11, l of everything below 2^-16 is subnormal, and the error stays at 2^-39: a reduction element 2^30 times the others and zero on the
// other side took all but nine of their bits.)  Of the four products of two elements h h', h l' and l h' are computed, each exact in the
// multiplier, and added up in fp32; |2^-11 l| is at most 2^-11 of x, so what the fourth would add is at most 2^-22 of the product.  Three
// instructions take the place of the six of three bf16 slices (gemm_split.h), with operands of four bytes an element, as many as fp32 has.
//
// Rows that hold an infinity or a NaN cannot be split.  They carry kNotFinite for their exponent, and a tile that meets one
// computes itself with the fp32 instruction from the operands as they were.
#pragma once

#include "gemm_core.h"
#include "internal.h"

#include <utility>

namespace tf {
namespace gemm {
namespace pair {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int BK = 16;                       // reduction elements a step: one matrix instruction's
constexpr int kFragment = 1024;              // bytes: 32 rows x 16 reduction elements of fp16, in the order of a wave's lanes
constexpr int kStepBytes = 2 * kFragment;    // of 32 rows: h, then l
constexpr int kNotFinite = INT32_MIN / 4;    // an exponent no finite row has

constexpr float kLowScale = 0x1p11f, kLowUnscale = 0x1p-11f;  // of l, of the sums of products with one

// A split operand: [block of 32 rows][step][h, l], the reduction padded with zeros to an even number of steps and the
// rows to whole blocks; value = (h + l kLowUnscale) * 2^-exps[row].
struct Packed {
  const char *planes;
  const int *exps;
  int blocks, steps;
};

// Work of a launch: tiles_m x tiles_n tiles, each by `pieces` workgroups over steps_per_piece steps, an even number.  B may be two operands
// of `blocks` blocks one behind the other, of which tiles number half_tiles each from the `first_half`-th on.
struct Work {
  int tiles_m, tiles_n, half_tiles, first_half, pieces, steps_per_piece;
  float *scratch;     // [tile][piece][BM * BN], pieces > 1
  unsigned *tickets;  // one a tile, zero before and after
};

template <int N, class F, int... I>
__device__ __forceinline__ void static_for_impl(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F &&f) {
  static_for_impl<N>(f, std::make_integer_sequence<int, N>{});
}

// A lane's part of a fragment.
__device__ inline f16x8 fragment(const char *at) { return *reinterpret_cast<const f16x8 *>(at); }

// The tile with the fp32 instruction, out of `a(row, k)` and `b(half, row, k)`: a stage is summed apart, as in gemm_split.h.
template <int BM, int BN, int TM, int TN, class ExactA, class ExactB>
__device__ __forceinline__ void exact_tile(f32x16 (&acc)[TM][TN], float *lds, const ExactA &a, const ExactB &b, int half,
                                           int m0, int n0, int k_begin, int k_end, int m_wave, int n_wave, int tid) {
  constexpr int STEP = 16, LDA = BM + 4, LDB = BN + 4;
  const int lane = tid & 63, lhalf = lane >> 5, lcol = lane & 31;
#pragma unroll 1
  for (int k0 = k_begin; k0 < k_end; k0 += STEP) {
    __syncthreads();
#pragma unroll 1
    for (int e = tid; e < BM * STEP; e += THREADS) {
      const int d = ExactA::kAlongRows ? e % BM : e / STEP, k = ExactA::kAlongRows ? e / BM : e % STEP;
      lds[k * LDA + d] = a(m0 + d, k0 + k);
    }
#pragma unroll 1
    for (int e = tid; e < BN * STEP; e += THREADS) {
      const int d = ExactB::kAlongRows ? e % BN : e / STEP, k = ExactB::kAlongRows ? e / BN : e % STEP;
      lds[STEP * LDA + k * LDB + d] = b(half, n0 + d, k0 + k);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        f32x16 sum;
#pragma unroll
        for (int v = 0; v < 16; ++v) sum[v] = 0.f;
#pragma unroll
        for (int k = 0; k < STEP; k += 2)
          sum = __builtin_amdgcn_mfma_f32_32x32x2f32(lds[(k + lhalf) * LDA + m_wave + 32 * i + lcol],
                                                     lds[STEP * LDA + (k + lhalf) * LDB + n_wave + 32 * j + lcol], sum, 0, 0, 0);
        acc[i][j] += sum;
      }
  }
}

// Four waves, 2 x 2 over a tile of 128 x 128, two workgroups a CU.  SLOTS steps of both operands in LDS, filled by loads that go
// there directly, and the operands of two steps in registers: while a step is multiplied, those of the next one are read from
// LDS and the step SLOTS further on is fetched to the slot that this step was read from, so that a fetch has
// SLOTS - 2 steps of time and no product waits for LDS.
//
// What bounds it is power, as for three slices: 4096^3 takes 334 us (411 TFLOP/s, 1 230 of the fp16 instruction; gemm_split.h
// 690), and on 256 x 256 and 256 x 128 tiles, which fetch half and three quarters as many bytes from L2, 322 and 334;
// 1024 x 8192 x 4096 167, 230 and 164, 4096 x 8192 x 1024 202, 199 and 227.  With one step under way instead of three 368 us.
constexpr int BM = 128, BN = 128, SLOTS = 4;
constexpr int BLOCKS = (BM + BN) / 32, SLOT = BLOCKS * kStepBytes, FETCHES = BLOCKS / 2;  // fetches: a wave's a step
//
// A launch may be two products: the workgroups of the second stand behind those of the first.
template <class Epilogue, class ExactA, class ExactB>
struct Product {
  Packed A, B;
  Work work;
  Epilogue ep;
  ExactA exact_a;
  ExactB exact_b;
  __host__ __device__ int groups() const { return work.tiles_m * work.tiles_n * work.pieces; }
};
template <class Products>
__global__ __launch_bounds__(THREADS, 2) void gemm_kernel(const Products products) {
  const bool is_second = Products::kCount > 1 && (int)blockIdx.x >= products.p[0].groups();
  const auto &product = products.p[is_second];
  const Packed A = product.A, B = product.B;
  const Work work = product.work;
  const int group = (int)blockIdx.x - (is_second ? products.p[0].groups() : 0);
  constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 32, TN = WN / 32;
  static_assert(SLOTS * SLOT >= 16 * (BM + 4 + BN + 4) * 4, "the fp32 pass reuses the slots");
  __shared__ __align__(16) char lds[SLOTS * SLOT];
  __shared__ unsigned flag;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m_wave = wave % 2 * WM, n_wave = wave / 2 * WN;
  const int tiles = work.tiles_m * work.tiles_n;
  // An XCD's tiles are neighbours in both directions, runs of eight tile rows of one tile column after the other: its L2 then
  // fetches a quarter of A and half of B of 4096 x 1024 x 8192, not all of A and an eighth of B.
  constexpr int RUN = 8;
  const int logical = xcd_contiguous(group, tiles * work.pieces);
  const int tile = logical % tiles, piece = logical / tiles;
  const int run = tile / (RUN * work.tiles_n), in_run = tile % (RUN * work.tiles_n), run_rows = min(RUN, work.tiles_m - run * RUN);
  const int tile_n = in_run / run_rows;
  const int half = work.first_half + tile_n / work.half_tiles;
  const int mb = (run * RUN + in_run % run_rows) * (BM / 32), nb = tile_n % work.half_tiles * (BN / 32);  // first blocks of 32 rows
  const int b_first = half * B.blocks;  // of the half
  const int s_begin = piece * work.steps_per_piece, s_end = min(A.steps, s_begin + work.steps_per_piece);

  if (tid == 0) flag = 0u;
  __syncthreads();
  {  // rows that cannot be split
    bool found = false;
    for (int r = tid; r < BM; r += THREADS) found |= A.exps[min(mb + r / 32, A.blocks - 1) * 32 + r % 32] == kNotFinite;
    for (int r = tid; r < BN; r += THREADS) found |= B.exps[(b_first + min(nb + r / 32, B.blocks - 1)) * 32 + r % 32] == kNotFinite;
    if (found) flag = 1u;
  }

  f32x16 acc[TM][TN], low[TM][TN];  // sums of h h', and of h l' + l h'
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = low[i][j][v] = 0.f;

  // Of a step's 2 BLOCKS fragments a wave fetches every fourth.  Blocks behind the operand's last one repeat it; what
  // comes of them is not stored.  Steps behind the end repeat the last one and are not read.  The load is written out
  // because the compiler takes every read of LDS for a reader of the loads into it that are under way, whichever slot they go to, and
  // waits for them; `arrived` is the wait that they need.  They write no register, and nothing else here goes by m0.
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + (uint32_t)wave * kFragment;
  const uint32_t lane_at = (uint32_t)lane * 16u + (uint32_t)(wave & 1) * kFragment;
  const size_t block_bytes = (size_t)A.steps * kStepBytes;
  auto fetch = [&](auto fetch_c, int s, int slot) {
    constexpr int t = 2 * decltype(fetch_c)::value;
    const int block = t + (wave >> 1);
    const char *from = t < BM / 32 ? A.planes + (size_t)min(mb + block, A.blocks - 1) * block_bytes
                                   : B.planes + (size_t)(b_first + min(nb + block - BM / 32, B.blocks - 1)) * block_bytes;
    from += (size_t)min(s, A.steps - 1) * kStepBytes;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_at + (uint32_t)(slot + t * kStepBytes)), lane_off = lane_at;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(lane_off), "s"(from));
  };
  f16x8 a[2][2][TM], b[2][2][TN];  // [step's parity][h, l]
  const char *const a_at = lds + m_wave / 32 * kStepBytes + lane * 16;
  const char *const b_at = lds + (BM + n_wave) / 32 * kStepBytes + lane * 16;
  constexpr int READS = 2 * (TM + TN), MFMAS = 3 * TM * TN;
  // the r-th operand of a step: those of the products that come first first
  auto read = [&](auto parity_c, auto read_c, int slot) {
    constexpr int h = decltype(parity_c)::value, r = decltype(read_c)::value, p = r / (TM + TN), i = r % (TM + TN);
    if constexpr (i < TM) a[h][p][i] = fragment(a_at + slot + i * kStepBytes + p * kFragment);
    else b[h][p][i - TM] = fragment(b_at + slot + (i - TM) * kStepBytes + p * kFragment);
  };
  auto multiply = [&](auto parity_c, auto index_c) {
    constexpr int h = decltype(parity_c)::value, n = decltype(index_c)::value;
    constexpr int p = n / (TM * TN), i = n % (TM * TN) / TN, j = n % TN, qa = p == 2, qb = p == 1;
    auto &sum = p == 0 ? acc : low;
    sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[h][qa][i], b[h][qb][j], sum[i][j], 0, 0, 0);
  };
  // everything that this wave has read from LDS has arrived, and of what it has fetched all but the last `under_way`, in all waves
  auto arrived = [](auto under_way) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(under_way)::value) : "memory");
  };
  std::integral_constant<int, (SLOTS - 2) * FETCHES> later;
  std::integral_constant<int, 0> none;
  // Step s out of registers; `slot` is where it was read from, `next` where the next step lies.  The reads and fetches stand evenly
  // between the products.
  auto step = [&](auto parity_c, int s, int slot, int next) {
    constexpr int h = decltype(parity_c)::value;
    static_for<MFMAS>([&](auto n_c) {
      constexpr int n = decltype(n_c)::value;
      static_for<READS>([&](auto r_c) {
        if constexpr (decltype(r_c)::value * MFMAS / READS == n) read(std::integral_constant<int, 1 - h>{}, r_c, next);
      });
      static_for<FETCHES>([&](auto t_c) {
        if constexpr (decltype(t_c)::value * MFMAS / FETCHES == n) fetch(t_c, s + SLOTS, slot);
      });
      multiply(parity_c, n_c);
      __builtin_amdgcn_sched_barrier(0);
    });
    arrived(later);
  };
  auto behind = [](int slot) { return slot + SLOT == SLOTS * SLOT ? 0 : slot + SLOT; };

  static_for<SLOTS>([&](auto slot_c) {
    constexpr int slot = decltype(slot_c)::value;
    static_for<FETCHES>([&](auto t_c) { fetch(t_c, s_begin + slot, slot * SLOT); });
  });
  arrived(later);  // the first two steps
  const bool exact = flag != 0u;  // uniform
  if (!exact) {
    std::integral_constant<int, 0> even;
    std::integral_constant<int, 1> odd;
    static_for<READS>([&](auto r_c) { read(even, r_c, 0); });
    // `arrived` stands between the reads of a slot and the fetches that refill it
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    int slot = 0;
    for (int s = s_begin; s < s_end; s += 2) {
      const int next = behind(slot), after = behind(next);
      step(even, s, slot, next);
      step(odd, s + 1, next, after);
      slot = after;
    }
    arrived(none);  // the fetches behind the end have landed
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] += low[i][j] * kLowUnscale;
  } else {
    arrived(none);
    exact_tile<BM, BN>(acc, reinterpret_cast<float *>(lds), product.exact_a, product.exact_b, half, mb * 32, nb * 32, s_begin * BK, s_end * BK,
                       m_wave, n_wave, tid);
  }

  if (work.pieces > 1) {  // the last piece of the tile to get here adds all of them, in their order (gemm_core.h: Fold)
    constexpr int SC1 = 16;
    constexpr uint32_t kPieceBytes = (uint32_t)(BM * BN) * 4u;
    const __amdgpu_buffer_rsrc_t pieces =
        make_rsrc(work.scratch + (size_t)tile * work.pieces * (BM * BN), (uint32_t)work.pieces * kPieceBytes);
    auto offset = [&](int p, int i, int j, int q) {
      return (int)((uint32_t)p * kPieceBytes + (uint32_t)((i * TN + j) * 4 + q) * (THREADS * 16u) + (uint32_t)tid * 16u);
    };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4v v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          __builtin_amdgcn_raw_buffer_store_b128(
              __builtin_bit_cast(__attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned, v), pieces,
              offset(piece, i, j, q), 0, SC1);
        }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) flag = atomicAdd(work.tickets + tile, 1u) == (unsigned)(work.pieces - 1) ? 2u : 3u;
    __syncthreads();
    if (flag != 2u) return;
    // 16 loads of a lane under way: they come from memory
    constexpr int BATCH = 16;
#pragma unroll
    for (int first = 0; first < TM * TN * 4; first += BATCH) {
      f32x4v sum[BATCH];
      for (int p = 0; p < work.pieces; ++p) {
        f32x4v v[BATCH];
#pragma unroll
        for (int e = 0; e < BATCH; ++e)
          v[e] = __builtin_bit_cast(f32x4v, __builtin_amdgcn_raw_buffer_load_b128(pieces, offset(p, 0, 0, first + e), 0, SC1));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < BATCH; ++e) sum[e] = p == 0 ? v[e] : sum[e] + v[e];
      }
#pragma unroll
      for (int e = 0; e < BATCH; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[(first + e) / 4 / TN][(first + e) / 4 % TN][4 * ((first + e) % 4) + c] = sum[e][c];
    }
    if (tid == 0) work.tickets[tile] = 0u;
  }

  // Exponents: those of this lane's columns, and of four rows at a time
  const auto state = product.ep.begin(mb * 32, half);
  int eb[TN];
  const int lhalf = lane >> 5, lcol = lane & 31;
#pragma unroll
  for (int j = 0; j < TN; ++j) eb[j] = exact ? 0 : -B.exps[(b_first + min(nb + n_wave / 32 + j, B.blocks - 1)) * 32 + lcol];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int block = mb + m_wave / 32 + i, row = 8 * q + 4 * lhalf;
      i32x4 ea = {0, 0, 0, 0};
      if (!exact) ea = *reinterpret_cast<const i32x4 *>(A.exps + min(block, A.blocks - 1) * 32 + row);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) v[j] = __builtin_ldexpf(acc[i][j][4 * q + e], eb[j] - ea[e]);
        product.ep.template store<TN>(state, m_wave + 32 * i + row + e, nb + n_wave / 32, lcol, v);
      }
    }
}

}  // namespace pair
}  // namespace gemm
}  // namespace tf
