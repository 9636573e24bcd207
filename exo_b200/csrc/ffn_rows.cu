// Feed-forward operators, the memory-bound passes: quantisation of rows, and the elementwise part of the gated
// projections' backward pass.
#include "ffn.cuh"

namespace exob200 {
namespace ffn {
namespace {

template <class E>
__global__ void __launch_bounds__(256) quantize_rows_kernel(int64_t K, const E* X, int8_t* Q, float* scale) {
  const E* x = X + (int64_t)blockIdx.x * K;
  int8_t* q = Q + (int64_t)blockIdx.x * K;
  __shared__ unsigned warp_top[8];
  // magnitudes compare like their bit patterns, and a NaN's is above infinity's
  unsigned top = 0;
  for (int64_t k = threadIdx.x; k < K; k += 256) top = max(top, __float_as_uint(fabsf(float(x[k]))));
  top = __reduce_max_sync(0xffffffffu, top);
  if (threadIdx.x % 32 == 0) warp_top[threadIdx.x / 32] = top;
  __syncthreads();
  for (int w = 0; w < 8; w++) top = max(top, warp_top[w]);
  const bool finite = top < 0x7f800000u;
  const float t = __uint_as_float(top);
  // 127 / top leaves fp32's range below 2^-121: such a row goes through with its values and top times 2^100
  const float up = t < 0x1p-100f ? 0x1p100f : 1.0f;
  const float inverse = finite && top ? __fdiv_rn(127.0f, t * up) : 0.0f;
  if (threadIdx.x == 0) scale[blockIdx.x] = finite ? __fdiv_rn(t, 127.0f) : __uint_as_float(0x7fffffffu);
  for (int64_t k = threadIdx.x; k < K; k += 256) {
    // adding 1.5 * 2^23 in the same rounding leaves the nearest integer in the low bits
    const float r = fmaf(float(x[k]) * up, inverse, 12582912.0f);
    q[k] = finite ? (int8_t)(__float_as_uint(r) & 0xff) : (int8_t)0;
  }
}

template <int ACT>
__global__ void __launch_bounds__(256)
gate_backward_kernel(int64_t n, const __nv_bfloat16* G, const __nv_bfloat16* U, const __nv_bfloat16* dH,
                     __nv_bfloat16* dG, __nv_bfloat16* dU) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const float g = __bfloat162float(G[i]), u = __bfloat162float(U[i]), d = __bfloat162float(dH[i]);
    const float p = gate_p<ACT>(g);
    dG[i] = __float2bfloat16_rn(d * u * gate_slope<ACT>(g, p));
    dU[i] = __float2bfloat16_rn(d * (g * p));
  }
}

}  // namespace

cudaError_t launch_quantize_rows(exo_b200_Context* ctx, int64_t M, int64_t K, const void* X, bool bf16, int8_t* Q,
                                 float* scale) {
  if (bf16)
    quantize_rows_kernel<<<(unsigned)M, 256, 0, ctx->stream>>>(K, static_cast<const __nv_bfloat16*>(X), Q, scale);
  else
    quantize_rows_kernel<<<(unsigned)M, 256, 0, ctx->stream>>>(K, static_cast<const float*>(X), Q, scale);
  return cudaGetLastError();
}

cudaError_t launch_gate_backward(exo_b200_Context* ctx, int act, int64_t n, const uint16_t* G, const uint16_t* U,
                                 const uint16_t* dH, uint16_t* dG, uint16_t* dU) {
  auto b = [](const uint16_t* q) { return reinterpret_cast<const __nv_bfloat16*>(q); };
  auto w = [](uint16_t* q) { return reinterpret_cast<__nv_bfloat16*>(q); };
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, (int64_t)ctx->sm_count * 8);
  if (act == EXO_B200_ACT_SILU)
    gate_backward_kernel<EXO_B200_ACT_SILU><<<grid, 256, 0, ctx->stream>>>(n, b(G), b(U), b(dH), w(dG), w(dU));
  else if (act == EXO_B200_ACT_GELU)
    gate_backward_kernel<EXO_B200_ACT_GELU><<<grid, 256, 0, ctx->stream>>>(n, b(G), b(U), b(dH), w(dG), w(dU));
  else
    gate_backward_kernel<EXO_B200_ACT_GELU_TANH><<<grid, 256, 0, ctx->stream>>>(n, b(G), b(U), b(dH), w(dG), w(dU));
  return cudaGetLastError();
}

}  // namespace ffn
}  // namespace exob200
