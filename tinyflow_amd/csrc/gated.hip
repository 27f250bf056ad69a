// Gated feed-forward product, forward and backward (no counterpart in the reference).
//
//   g = x Wg, u = x Wu, h = act(g) u        x [M, K], Wg and Wu [K, F]
//   dg = dh u act'(g), du = dh act(g);  dx = dg Wg^T + du Wu^T,  dWg = x^T dg,  dWu = x^T du
#include "internal.h"

#include <algorithm>

using namespace tf;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4u __attribute__((aligned(4)));
constexpr int kThreads = 256;

enum Activation { kSigmoid = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// v_rcp_f32 is right to one step of the last place
__device__ inline float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + expf(-g)); }

template <int ACT>
__device__ inline float act_of(float g) {
  if (ACT == kRelu) return g > 0.f ? g : g != g ? g : 0.f;
  if (ACT == kGelu) return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
  const float s = sigmoid(g);
  return ACT == kSigmoid ? s : g * s;
}

// act(g) and act'(g)
template <int ACT>
__device__ inline void act_and_slope(float g, float &act, float &slope) {
  if (ACT == kRelu) {
    act = act_of<kRelu>(g);
    slope = g > 0.f ? 1.f : 0.f;
  } else if (ACT == kGelu) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    act = g * cdf;
    slope = cdf + g * (0.39894228040143268f * expf(-0.5f * g * g));
  } else {
    const float s = sigmoid(g);
    act = ACT == kSigmoid ? s : g * s;
    slope = ACT == kSigmoid ? s * (1.f - s) : s * (1.f + g * (1.f - s));
  }
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

// Bound by HBM: 12 and 20 bytes an element.
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

unsigned vectors_grid(int64_t count) { return (unsigned)((count + 4 * kThreads - 1) / (4 * kThreads)); }

bool is_pair(const DLArray *pre, const DLArray *one) {
  return pre->ndim == one->ndim + 1 && pre->shape[0] == 2 &&
         std::equal(one->shape, one->shape + one->ndim, pre->shape + 1);
}

struct View {
  int64_t shape[2];
  DLArray array;
  View(float *data, int64_t rows, int64_t cols, DLContext ctx) : shape{rows, cols}, array{data, ctx, 2, shape} {}
};

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
  TF_REQUIRE(n < (int64_t)1 << 40, "too many elements");
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
  TF_REQUIRE(n < (int64_t)1 << 40, "too many elements");
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
  TF_REQUIRE(!being_captured(s), "the call takes scratch, which a captured stream cannot give back");
  if (M == 0 || F == 0) return 0;
  float *p = pre ? (float *)pre->data : (float *)device_alloc((size_t)M * F * 8, s);
  if (!p) {
    if (memorytoSaving) *memorytoSaving = shortfall(block_bytes((size_t)M * F * 8));
    return 0;
  }
  View g(p, M, F, input->ctx), u(p + M * F, M, F, input->ctx);
  int rc = DLGpuMatrixMultiply(input, false, gate, false, &g.array, nullptr, stream);
  if (rc == 0) rc = DLGpuMatrixMultiply(input, false, up, false, &u.array, nullptr, stream);
  if (rc == 0 && output)
    with_activation(activation, [&](auto act) {
      hipLaunchKernelGGL(activation_kernel<decltype(act)::value>, dim3(vectors_grid(M * F)), dim3(kThreads), 0, s, p, p + M * F,
                         (float *)output->data, M * F);
    });
  if (!pre) device_free(p, s);
  return rc != 0 ? rc : finish(s, "DLGpuGatedFeedForward");
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
  const size_t bytes = ((pre ? (size_t)M * F * 2 : 0) + (dinput ? (size_t)M * K : 0)) * 4;
  float *scratch = (float *)device_alloc(bytes, s);
  if (!scratch) {
    if (memorytoSaving) *memorytoSaving = shortfall(block_bytes(bytes));
    return 0;
  }
  float *d = pre ? scratch : (float *)doutput->data;
  if (pre && M * F > 0)
    with_activation(activation, [&](auto act) {
      const float *g = (const float *)pre->data;
      hipLaunchKernelGGL(activation_backward_kernel<decltype(act)::value>, dim3(vectors_grid(M * F)), dim3(kThreads), 0, s, g,
                         g + M * F, (const float *)doutput->data, d, d + M * F, M * F);
    });
  View dg(d, M, F, input->ctx), du(d + M * F, M, F, input->ctx);
  View other(scratch + (pre ? M * F * 2 : 0), M, K, input->ctx);
  int rc = 0;
  if (dinput) {
    rc = DLGpuMatrixMultiply(&dg.array, false, gate, true, dinput, nullptr, stream);
    if (rc == 0) rc = DLGpuMatrixMultiply(&du.array, false, up, true, &other.array, nullptr, stream);
    if (rc == 0) rc = DLGpuMatrixElementwiseAdd(dinput, &other.array, dinput, stream);
  }
  if (rc == 0 && dgate) rc = DLGpuMatrixMultiply(input, true, &dg.array, false, dgate, nullptr, stream);
  if (rc == 0 && dup) rc = DLGpuMatrixMultiply(input, true, &du.array, false, dup, nullptr, stream);
  device_free(scratch, s);
  return rc != 0 ? rc : finish(s, "DLGpuGatedFeedForwardBackward");
}
