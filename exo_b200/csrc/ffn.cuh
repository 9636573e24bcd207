// Feed-forward operators (int8 products with token and channel scales, gated projections and their
// backward pass): what the entry points in ffn_api.cu hand to the kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace exob200 {
namespace ffn {

enum Kind {
  SCALED = 0,  // C[M,N] = (A[M,K] B[N,K]^T) * row_scale * col_scale + bias, int8 operands
  GATED,       // H[M,N] = act(A B0^T) * (A B1^T), bf16; G and U kept on request
  GATED_I8,    // the same on int8 operands with scales
  DGRAD,       // C[M,N] = A0[M,K] B0[K,N] + A1[M,K] B1[K,N], bf16
  WGRAD        // C0[M,N] = A0[K,M]^T B0[K,N], C1 = A1^T B0, bf16
};

// One product.  M, N: rows and columns of an output; K: the reduction length.  Device pointers.
struct Problem {
  int64_t M, N, K;
  const void *a0, *a1, *b0, *b1;
  const float *row_scale, *col_scale, *col_scale1, *bias;
  void *c0, *c1, *c2;
  int act;
};

// All are ordered on the context's stream.
cudaError_t launch_quantize_rows(exo_b200_Context* ctx, int64_t M, int64_t K, const void* X, bool bf16, int8_t* Q,
                                 float* scale);
// after_own_kernel: the kernel before this one on the stream belongs to the same call and was launched in the ordinary
// way (or waits for one that was), so this one may be scheduled before it ends.
cudaError_t launch_product(exo_b200_Context* ctx, Kind kind, bool out_f32, const Problem& p, bool after_own_kernel);
// dX = dG Wg + dU Wu [M,K] and dWg = dG^T X, dWu = dU^T X [F,K], each only where it is wanted (dWg and dWu together);
// after launch_gate_backward on the same stream.  dG and dU enter as rounded to bf16, the type that the tensor core
// multiplies: the gradients are 2.3e-3 of their norm from exact, 1.7e-3 of it their own rounding.  Entering unrounded, as
// sums of two bf16 numbers, they would come to 1.7e-3 for twice the products (a training step's backward pass of 8192 x
// 8192 x 4096 is 1.6 ms of products in 1.7).
cudaError_t launch_gradients(exo_b200_Context* ctx, int64_t M, int64_t F, int64_t K, const void* X, const void* Wg,
                             const void* Wu, const void* dG, const void* dU, void* dX, void* dWg, void* dWu);
// The products of a few rows (ffn_gemv.cu): whether they are taken for a problem, and their launch.
constexpr int kRowTokenBytes = 96 * 1024;  // tokens that a CTA keeps in shared memory
bool rows_wanted(Kind kind, const Problem& p);
cudaError_t launch_rows(exo_b200_Context* ctx, Kind kind, bool out_f32, const Problem& p, bool after_own_kernel);
// The same with the quantisation of the tokens X (bf16, or fp32 where the output is) in the one kernel; p.a0 and
// p.row_scale are written.
bool linear_rows_wanted(const Problem& p, bool f32);
cudaError_t launch_linear_rows(exo_b200_Context* ctx, bool f32, const Problem& p, const void* X);
// dG = dH * U * act'(G), dU = dH * act(G), n elements
cudaError_t launch_gate_backward(exo_b200_Context* ctx, int act, int64_t n, const uint16_t* G, const uint16_t* U,
                                 const uint16_t* dH, uint16_t* dG, uint16_t* dU);

// ------------------------------------------------------------------ activations
// All three are g * p(g) with p the logistic function of g, the normal distribution function, or the logistic
// function of twice the tanh argument ((1 + tanh z) / 2 = 1 / (1 + exp(-2 z))).  The fast exponential's error is 2^-22
// and its argument's rounding, which grows to 5e-6 at the end of fp32's range; with the argument's own roundings p is
// within 2^-13 of itself wherever it is above 2^-126 (below, the fast division gives zero), far inside the bf16 rounding
// of every result.
__device__ __forceinline__ float logistic(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

constexpr float kRoot2Pi = 0.79788456f;       // sqrt(2 / pi)
constexpr float kTanhCubic = 0.044715f;
// beyond this p is 0 or 1 in fp32 for the two GELUs; keeps the cubic and its derivative finite
constexpr float kGeluClamp = 32.0f;
// g between -kGeluClamp and kGeluClamp.  A NaN stays one (fminf and fmaxf take the other operand in its place).
__device__ __forceinline__ float clamped_gate(float g) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(g), "f"(-kGeluClamp));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(c) : "f"(kGeluClamp));
  return c;
}

// The normal distribution function: Phi(-x) = exp(-x^2 / 2) t (c1 + c2 t + ... + c6 t^5) with t = 1 / (1 + p x), the form
// of formula 7.1.26 in Abramowitz and Stegun's Handbook of Mathematical Functions, which bounds the absolute error (its
// own coefficients are 1 % off at g = -8).  These were fitted, as a linear program over 0 <= x <= 14, to be close
// relatively: within 9e-7 for x < 1, 2.6e-5 in the tail, 2e-7 absolutely.  In fp32 the square and the exponential add
// 2e-5 at x = 13; half a step of bf16 is 2e-3 to 4e-3.  The sixth coefficient costs 2 % where the epilogue counts
// (1000 x 4096 x 512 gated, G and U kept: 18.2 us, 17.7 with the formula's own five; erfcf is three times as long).
__device__ __forceinline__ float normal_cdf(float g) {
  const float t = __fdividef(1.0f, 1.0f + 0.29658739f * fabsf(g));
  float y = fmaf(t, -0.082954542f, 0.243579873f);
  y = fmaf(t, y, -0.046016811f);
  y = fmaf(t, y, 0.157158702f);
  y = fmaf(t, y, 0.109263362f);
  y = fmaf(t, y, 0.118969216f);
  y = y * t * __expf(-0.5f * g * g);
  return g < 0.0f ? y : 1.0f - y;
}

template <int ACT>
__device__ __forceinline__ float gate_p(float g) {
  if (ACT == EXO_B200_ACT_SILU) return logistic(g);
  if (ACT == EXO_B200_ACT_GELU) return normal_cdf(g);
  const float c = clamped_gate(g);
  return logistic(2.0f * kRoot2Pi * (c + kTanhCubic * c * c * c));
}
template <int ACT>
__device__ __forceinline__ float gate(float g) {
  return g * gate_p<ACT>(g);
}
// derivative of g p(g), given p
template <int ACT>
__device__ __forceinline__ float gate_slope(float g, float p) {
  if (ACT == EXO_B200_ACT_SILU) return p * (1.0f + g * (1.0f - p));
  if (ACT == EXO_B200_ACT_GELU) return p + g * __expf(-0.5f * g * g) * (0.5f * kRoot2Pi);
  const float c = clamped_gate(g);
  return p + c * p * (1.0f - p) * (2.0f * kRoot2Pi) * (1.0f + 3.0f * kTanhCubic * c * c);
}

__device__ __forceinline__ float scaled(int32_t acc, float row, float col) {
  return __int2float_rn(acc) * row * col;
}

// ------------------------------------------------------------------ quantisation of a row
// Magnitudes compare like their bit patterns, and a NaN's is above infinity's.
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(fabsf(x)); }

struct Step {
  float inverse, up;  // q = nearest integer to (x * up) * inverse
  bool finite;
  float scale;
};
__device__ __forceinline__ Step step_of(unsigned top) {
  Step s;
  s.finite = top < 0x7f800000u;
  const float t = __uint_as_float(top);
  // 127 / top leaves fp32's range below 2^-121: such a row goes through with its values and top times 2^100
  s.up = t < 0x1p-100f ? 0x1p100f : 1.0f;
  s.inverse = s.finite && top ? __fdiv_rn(127.0f, t * s.up) : 0.0f;
  s.scale = s.finite ? __fdiv_rn(t, 127.0f) : __uint_as_float(0x7fffffffu);
  return s;
}
// Adding 1.5 * 2^23 in the same rounding as the product leaves the nearest integer in the low bits.
__device__ __forceinline__ uint32_t quantized(float x, const Step& s) {
  return s.finite ? __float_as_uint(fmaf(x * s.up, s.inverse, 12582912.0f)) & 0xffu : 0u;
}

template <class E>
__device__ __forceinline__ void widen(const uint4& v, float (&f)[16 / sizeof(E)]);
template <>
__device__ __forceinline__ void widen<float>(const uint4& v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
}
template <>
__device__ __forceinline__ void widen<__nv_bfloat16>(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; j++) {
    f[2 * j] = __uint_as_float(w[j] << 16);
    f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}

}  // namespace ffn
}  // namespace exob200
