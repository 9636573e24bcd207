// Feed-forward operators, plain CUDA-core kernels: 64 x 64 tiles through shared memory, four by four outputs
// for each thread.
#include "ffn.cuh"

namespace exob200 {
namespace ffn {
namespace {

constexpr int T = 64, TK = 16;

template <class E>
struct Sum {
  using type = float;
};
template <>
struct Sum<int8_t> {
  using type = int32_t;
};
__device__ __forceinline__ void mac(float& c, __nv_bfloat16 a, __nv_bfloat16 b) {
  c = fmaf(__bfloat162float(a), __bfloat162float(b), c);
}
__device__ __forceinline__ void mac(int32_t& c, int8_t a, int8_t b) { c += (int32_t)a * (int32_t)b; }

// s[k][i] = X[i0 + i, k0 + k] of an operand with element strides (si, sk); zero outside
template <class E>
__device__ __forceinline__ void load_tile(E (&s)[TK][T + 4], const E* X, int64_t i0, int64_t k0, int64_t I, int64_t K,
                                          int64_t si, int64_t sk) {
  for (int e = threadIdx.x; e < T * TK; e += 256) {
    // neighbouring threads along the contiguous direction
    const int i = sk == 1 ? e / TK : e % T, k = sk == 1 ? e % TK : e / T;
    s[k][i] = (i0 + i < I && k0 + k < K) ? X[(i0 + i) * si + (k0 + k) * sk] : E(0);
  }
}

template <int KIND, class E, class O, int ACT>
__global__ void __launch_bounds__(256) simt_kernel(Problem p) {
  constexpr bool TWO = KIND == GATED || KIND == GATED_I8;
  using S = typename Sum<E>::type;
  __shared__ E sa[TK][T + 4], sb[TK][T + 4], sb1[TWO ? TK : 1][T + 4];
  const int64_t i0 = (int64_t)blockIdx.x * T, j0 = (int64_t)blockIdx.y * T;
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  S acc[TWO ? 2 : 1][4][4] = {};
  const int halves = KIND == DGRAD ? 2 : 1;
  for (int h = 0; h < halves; h++) {
    const E* A = static_cast<const E*>(h || (KIND == WGRAD && blockIdx.z) ? p.a1 : p.a0);
    const E* B = static_cast<const E*>(h ? p.b1 : p.b0);
    for (int64_t k0 = 0; k0 < p.K; k0 += TK) {
      if (KIND == WGRAD)
        load_tile(sa, A, i0, k0, p.M, p.K, 1, p.M);
      else
        load_tile(sa, A, i0, k0, p.M, p.K, p.K, 1);
      if (KIND == WGRAD || KIND == DGRAD)
        load_tile(sb, B, j0, k0, p.N, p.K, 1, p.N);
      else
        load_tile(sb, B, j0, k0, p.N, p.K, p.K, 1);
      if constexpr (TWO) load_tile(sb1, static_cast<const E*>(p.b1), j0, k0, p.N, p.K, p.K, 1);
      __syncthreads();
      for (int k = 0; k < TK; k++)
        for (int i = 0; i < 4; i++)
          for (int j = 0; j < 4; j++) {
            mac(acc[0][i][j], sa[k][ti + i], sb[k][tj + j]);
            if constexpr (TWO) mac(acc[1][i][j], sa[k][ti + i], sb1[k][tj + j]);
          }
      __syncthreads();
    }
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const int64_t r = i0 + ti + i, c = j0 + tj + j, at = r * p.N + c;
      if (r >= p.M || c >= p.N) continue;
      if constexpr (KIND == SCALED) {
        const float v = scaled(acc[0][i][j], p.row_scale[r], p.col_scale[c]) + (p.bias ? p.bias[c] : 0.f);
        static_cast<O*>(p.c0)[at] = O(v);
      } else if constexpr (TWO) {
        float g, u;
        if constexpr (KIND == GATED_I8) {
          g = scaled(acc[0][i][j], p.row_scale[r], p.col_scale[c]);
          u = scaled(acc[1][i][j], p.row_scale[r], p.col_scale1[c]);
        } else {
          g = acc[0][i][j];
          u = acc[1][i][j];
        }
        static_cast<O*>(p.c0)[at] = O(gate<ACT>(g) * u);
        if (p.c1) {
          static_cast<O*>(p.c1)[at] = O(g);
          static_cast<O*>(p.c2)[at] = O(u);
        }
      } else {
        static_cast<O*>(KIND == WGRAD && blockIdx.z ? p.c1 : p.c0)[at] = O(acc[0][i][j]);
      }
    }
}

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

template <int KIND, class E, class O, int ACT>
cudaError_t go(exo_b200_Context* ctx, const Problem& p) {
  const dim3 grid((unsigned)((p.M + T - 1) / T), (unsigned)((p.N + T - 1) / T), KIND == WGRAD ? 2 : 1);
  if (grid.y > 65535) return cudaErrorInvalidValue;
  simt_kernel<KIND, E, O, ACT><<<grid, 256, 0, ctx->stream>>>(p);
  return cudaGetLastError();
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

cudaError_t launch_product(exo_b200_Context* ctx, Kind kind, bool out_f32, const Problem& p) {
  using bf16 = __nv_bfloat16;
  switch (kind) {
    case SCALED:
      return out_f32 ? go<SCALED, int8_t, float, 0>(ctx, p) : go<SCALED, int8_t, bf16, 0>(ctx, p);
    case GATED:
      return p.act == 0 ? go<GATED, bf16, bf16, 0>(ctx, p)
             : p.act == 1 ? go<GATED, bf16, bf16, 1>(ctx, p)
                          : go<GATED, bf16, bf16, 2>(ctx, p);
    case GATED_I8:
      return p.act == 0 ? go<GATED_I8, int8_t, bf16, 0>(ctx, p)
             : p.act == 1 ? go<GATED_I8, int8_t, bf16, 1>(ctx, p)
                          : go<GATED_I8, int8_t, bf16, 2>(ctx, p);
    case DGRAD:
      return go<DGRAD, bf16, bf16, 0>(ctx, p);
    default:
      return go<WGRAD, bf16, bf16, 0>(ctx, p);
  }
}

}  // namespace ffn
}  // namespace exob200
