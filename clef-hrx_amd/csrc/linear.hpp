// Products of bf16 rows and bf16 weights with an epilogue: arguments and the
// device helpers that the kernels share.
//   y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n]
//   h[m][n] = act(gate sum + gate bias) * (up sum + up bias)      (gate/up)
// Everything is f32 up to the one rounding of the output (none for f32).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"
#include "gemm_dma.hpp"
#include "launch.hpp"

namespace clef {

enum LinearAct { kActNone, kActRelu, kActGelu, kActGeluTanh, kActSilu, kActSigmoid, kActs };

struct LinearArgs {
  const uint16_t* x;  // [m][k], rows x_stride elements apart
  int64_t m, x_stride;
  int n, k;
  const uint16_t* w;   // [n][k], rows w_stride apart
  const uint16_t* w2;  // gate/up: the up weight
  int64_t w_stride;
  const void* bias;  // bf16 or f32 [n], or NULL
  const void* bias2;
  bool bias_f32;
  int act;
  const uint16_t* residual;  // bf16, rows residual_stride apart, or NULL
  int64_t residual_stride;
  void* out;  // bf16 or f32, rows out_stride apart
  int64_t out_stride;
  bool out_f32;
  // Products split along k: parts 1, or each part's sums go to partial (f32 [part]
  // [matrix][m][n rounded up to 4]) and another launch adds them
  int parts;
  float* partial;
};

// Scratch for the parts of a product whose operands' rows lie on 16 bytes, and for
// those of this one.
size_t linear_workspace_bytes(int64_t m, int n, int k, bool gate_up);
size_t linear_workspace_bytes(const LinearArgs& p, bool gate_up);
const char* linear_kernel_name(int64_t m, int n, int k, bool gate_up, bool aligned);
hipError_t launch_linear(LinearArgs p, bool gate_up, void* workspace, hipStream_t stream);

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// D = W A^T of a 16 x 16 tile over 32 k, added to c. Lane l holds weight row
// l % 16 in w and activation row l % 16 in a, eight values of k-group l / 16 (any
// order of k that both share); D's lane l holds activation row l % 16 and weight
// rows 4 (l / 16) .. + 3.
__device__ __forceinline__ v4f mfma_bf16(u4 w, u4 a, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, a), c, 0, 0,
                                                 0);
}

// 1 / (1 + exp(-v)): the hardware's exp2 and reciprocal, each within 1 ulp; the
// limits are the function's (exp2 of -inf is 0, 1 / inf is 0).
__device__ __forceinline__ float sigmoid_f32(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f));
}

// v Phi(v), Phi the normal distribution function: Phi(-a) = exp(-a^2 / 2) t P(t)
// for a >= 0 with t = 1 / (1 + 0.3 a), P of degree 7 fitted to erfcx(a / sqrt 2) /
// 2 (2.0e-7 of the value for a in 0 .. 14, the coefficients in f32). The tail keeps its
// relative accuracy (with the square's rounding 2.5e-6 up to a = 5), which 1 + erf(v)
// would lose.
__device__ __forceinline__ float gelu_f32(float v) {
  const float a = __builtin_fabsf(v), t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.3f, 1.0f));
  float p = 0.0356752909719944f;
  p = __builtin_fmaf(p, t, -0.15720513463020325f);
  p = __builtin_fmaf(p, t, 0.20635683834552765f);
  p = __builtin_fmaf(p, t, -0.05368649214506149f);
  p = __builtin_fmaf(p, t, 0.1285630166530609f);
  p = __builtin_fmaf(p, t, 0.0999131053686142f);
  p = __builtin_fmaf(p, t, 0.12075401097536087f);
  p = __builtin_fmaf(p, t, 0.11962929368019104f);
  const float q = p * t * __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);
  return v * (v < 0.0f ? q : 1.0f - q);
}

// Of every value; `act` is uniform. A tile's epilogue holds the bodies once per eight
// values, so the last three share one: v or 1 times sigmoid(v (a + b v^2)), b = 0 but
// for the tanh form of GELU, 0.5 v (1 + tanh(z)) = v sigmoid(2 z) with z = sqrt(2 /
// pi) (v + 0.044715 v^3). NaN stays NaN (ReLU too).
template <int N>
__device__ __forceinline__ void linear_act(v4f (&y)[N], int act) {
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) y[i][t] = f(y[i][t]);
  };
  if (act == kActNone) return;
  if (act == kActGelu) return each([](float v) { return gelu_f32(v); });
  if (act == kActRelu) return each([](float v) { return v < 0.0f ? 0.0f : v; });
  const float a = act == kActGeluTanh ? 1.59576912160573f : 1.0f, b = act == kActGeluTanh ? 0.0713548162726f : 0.0f;
  each([=](float v) {
    const float square = __builtin_fminf(v * v, 1e30f);  // (0 times infinity)
    const float s = sigmoid_f32(v * __builtin_fmaf(square, b, a));
    return act == kActSigmoid ? s : v * s;
  });
}

// Columns col .. + 3 of a bias, and of a residual row: loads of any alignment
// (one instruction), columns past the last are zeros.
__device__ __forceinline__ v4f linear_bias4(const void* bias, bool f32, int col, int n) {
  v4f v = {0, 0, 0, 0};
  if (!bias) return v;
  if (f32) {
    const float* from = static_cast<const float*>(bias) + col;
    if (col + 4 <= n) {
      __builtin_memcpy(&v, from, 16);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (col + t < n) v[t] = from[t];
    }
    return v;
  }
  const uint16_t* from = static_cast<const uint16_t*>(bias) + col;
  uint2 w = {0, 0};
  if (col + 4 <= n) {
    __builtin_memcpy(&w, from, 8);
  } else {
    if (col < n) w.x = from[0];
    if (col + 1 < n) w.x |= (uint32_t)from[1] << 16;
    if (col + 2 < n) w.y = from[2];
  }
  return v4f{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
}

// Eight bf16 of which `left` are inside the row (those past it are zeros; not stored).
__device__ __forceinline__ void linear_load8(const uint16_t* from, int left, uint2 (&v)[2]) {
  if (left >= 8) {
    __builtin_memcpy(v, from, 16);
    return;
  }
  uint32_t w[4] = {};
#pragma unroll
  for (int t = 0; t < 7; ++t)
    if (t < left) w[t / 2] |= (uint32_t)from[t] << (16 * (t % 2));
  v[0] = uint2{w[0], w[1]};
  v[1] = uint2{w[2], w[3]};
}

__device__ __forceinline__ void linear_store8(uint16_t* to, int left, const uint2 (&v)[2]) {
  if (left >= 8) {
    __builtin_memcpy(to, v, 16);
    return;
  }
  const uint32_t w[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
#pragma unroll
  for (int t = 0; t < 7; ++t)
    if (t < left) to[t] = (uint16_t)(w[t / 2] >> (16 * (t % 2)));
}

__device__ __forceinline__ v4f linear_residual4(const LinearArgs& p, int64_t row, int col) {
  return linear_bias4(p.residual + row * p.residual_stride, false, col, p.n);
}

// act(y + bias), and the product with the up sums for gate/up.
template <bool GU>
__device__ __forceinline__ v4f linear_finish4(const LinearArgs& p, v4f y, v4f bias, v4f y2, v4f bias2) {
  v4f v[1] = {y + bias};
  linear_act(v, p.act);
  if constexpr (GU) v[0] *= y2 + bias2;
  return v[0];
}

// Columns col .. + 3 of an output row, any alignment, those past the last left out.
__device__ __forceinline__ void linear_store4(const LinearArgs& p, int64_t row, int col, v4f y) {
  const int64_t at = row * p.out_stride + col;
  if (p.out_f32) {
    float* to = static_cast<float*>(p.out) + at;
    if (col + 4 <= p.n) {
      __builtin_memcpy(to, &y, 16);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (col + t < p.n) to[t] = y[t];
    }
    return;
  }
  uint16_t* to = static_cast<uint16_t*>(p.out) + at;
  const uint2 v = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
  if (col + 4 <= p.n) {
    __builtin_memcpy(to, &v, 8);
  } else {
    if (col < p.n) to[0] = (uint16_t)v.x;
    if (col + 1 < p.n) to[1] = (uint16_t)(v.x >> 16);
    if (col + 2 < p.n) to[2] = (uint16_t)v.y;
  }
}

// A part's sums of columns col .. + 3 (of matrix `which` of `matrices`).
__device__ __forceinline__ float* linear_partial4(const LinearArgs& p, int part, int which, int matrices, int64_t row,
                                                  int col) {
  const int64_t pitch = (p.n + 3) & ~3;
  return p.partial + (((int64_t)part * matrices + which) * p.m + row) * pitch + col;
}

// All of it: sums y (gate/up: y the gate's, y2 the up's) of one row.
template <bool GU>
__device__ __forceinline__ void linear_epilogue4(const LinearArgs& p, int64_t row, int col, v4f y, v4f y2) {
  v4f bias2 = {0, 0, 0, 0};
  if constexpr (GU) bias2 = linear_bias4(p.bias2, p.bias_f32, col, p.n);
  y = linear_finish4<GU>(p, y, linear_bias4(p.bias, p.bias_f32, col, p.n), y2, bias2);
  if (p.residual) y += linear_residual4(p, row, col);
  linear_store4(p, row, col, y);
}

}  // namespace

}  // namespace clef
