// Feed-forward operators, the memory-bound passes: quantisation of rows, and the elementwise part of the gated
// projections' backward pass.
#include "ffn.cuh"
#include "tc_common.cuh"

namespace exob200 {
namespace ffn {
namespace {

using tc::aligned16;
using umma::grid_dep_launch;

// ------------------------------------------------------------------ quantisation
// Largest of the magnitudes over the warp, or the CTA's eight warps, that share a row.
template <int WARPS>
__device__ __forceinline__ unsigned row_top(unsigned top) {
  top = __reduce_max_sync(0xffffffffu, top);
  if (WARPS > 1) {
    __shared__ unsigned warp_top[8];
    if (threadIdx.x % 32 == 0) warp_top[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = max(top, warp_top[w]);
  }
  return top;
}

// Rows that are whole 16-byte vectors: each is read once and stays in registers (V vectors a thread) between the search
// for its largest magnitude and the rounding.  Where rows are many and short, a warp takes one, with up to eight loads in
// flight and no one to agree with (8192 x 1024 fp32: 6.6 us, 10.8 with a CTA a row); otherwise a CTA (2048 x 4096 bf16:
// 4.8 us, 4.9 with two warps a row; 8192 x 8192 33 us, 6.1 TB/s, 38 with four).
template <class E, int V, int WARPS>
__global__ void __launch_bounds__(256) quantize_vectors_kernel(int64_t M, int K, const E* X, int8_t* Q, float* scale) {
  constexpr int N = 16 / sizeof(E);
  grid_dep_launch();
  const int64_t row = (int64_t)blockIdx.x * (8 / WARPS) + threadIdx.x / (32 * WARPS);
  if (row >= M) return;
  const int t = threadIdx.x % (32 * WARPS);
  const uint4* x = reinterpret_cast<const uint4*>(X + row * K);
  uint4 v[V];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int at = t + i * 32 * WARPS;
    v[i] = at * N < K ? x[at] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < V; i++) {
    float f[N];
    widen<E>(v[i], f);
#pragma unroll
    for (int j = 0; j < N; j++) top = max(top, magnitude(f[j]));
  }
  const Step s = step_of(row_top<WARPS>(top));
  if (t == 0) scale[row] = s.scale;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int at = t + i * 32 * WARPS;
    if (at * N >= K) break;
    float f[N];
    widen<E>(v[i], f);
    uint32_t w[N / 4] = {};
#pragma unroll
    for (int j = 0; j < N; j++) w[j / 4] |= quantized(f[j], s) << (8 * (j % 4));
    uint32_t* q = reinterpret_cast<uint32_t*>(Q + row * K) + at * (N / 4);
    if constexpr (N == 8)
      *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else
      *q = w[0];
  }
}

// Rows of any alignment, element by element but otherwise the same: up to V elements a thread, all on their way at once
// and kept (a loop over them waits for each: 1283 x 1446 fp32 10.2 us, 5.3 here).
template <class E, int V, int WARPS>
__global__ void __launch_bounds__(256) quantize_elements_kernel(int64_t M, int K, const E* X, int8_t* Q, float* scale) {
  grid_dep_launch();
  const int64_t row = (int64_t)blockIdx.x * (8 / WARPS) + threadIdx.x / (32 * WARPS);
  if (row >= M) return;
  const int t = threadIdx.x % (32 * WARPS);
  const E* x = X + row * K;
  int8_t* q = Q + row * K;
  float v[V];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int k = t + i * 32 * WARPS;
    v[i] = k < K ? float(x[k]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < V; i++) top = max(top, magnitude(v[i]));
  const Step s = step_of(row_top<WARPS>(top));
  if (t == 0) scale[row] = s.scale;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int k = t + i * 32 * WARPS;
    if (k < K) q[k] = (int8_t)quantized(v[i], s);
  }
}

// Rows too long for registers: a CTA a row, the second pass out of the caches.
template <class E>
__global__ void __launch_bounds__(256) quantize_rows_kernel(int64_t K, const E* X, int8_t* Q, float* scale) {
  grid_dep_launch();
  const E* x = X + (int64_t)blockIdx.x * K;
  int8_t* q = Q + (int64_t)blockIdx.x * K;
  unsigned top = 0;
#pragma unroll 8
  for (int64_t k = threadIdx.x; k < K; k += 256) top = max(top, magnitude(float(x[k])));
  const Step s = step_of(row_top<8>(top));
  if (threadIdx.x == 0) scale[blockIdx.x] = s.scale;
#pragma unroll 8
  for (int64_t k = threadIdx.x; k < K; k += 256) q[k] = (int8_t)quantized(float(x[k]), s);
}

template <class E>
cudaError_t quantize(exo_b200_Context* ctx, int64_t M, int64_t K, const E* X, int8_t* Q, float* scale) {
  constexpr int N = 16 / sizeof(E);  // elements of a vector
  const cudaStream_t st = ctx->stream;
  const bool vectors = K % N == 0 && aligned16(X) && reinterpret_cast<uintptr_t>(Q) % N == 0;
  const unsigned m = (unsigned)M;
  const bool many = M >= 8 * ctx->sm_count;
  if (vectors && many && K <= 128 * N)
    quantize_vectors_kernel<E, 4, 1><<<(m + 7) / 8, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (vectors && many && K <= 256 * N)
    quantize_vectors_kernel<E, 8, 1><<<(m + 7) / 8, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (vectors && K <= 256 * N)
    quantize_vectors_kernel<E, 1, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (vectors && K <= 512 * N)
    quantize_vectors_kernel<E, 2, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (vectors && K <= 1024 * N)
    quantize_vectors_kernel<E, 4, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (vectors && K <= 2048 * N)
    quantize_vectors_kernel<E, 8, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (vectors && K <= 4096 * N)
    quantize_vectors_kernel<E, 16, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (many && K <= 512)
    quantize_elements_kernel<E, 16, 1><<<(m + 7) / 8, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (K <= 2048)
    quantize_elements_kernel<E, 8, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (K <= 4096)
    quantize_elements_kernel<E, 16, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else if (K <= 8192)
    quantize_elements_kernel<E, 32, 8><<<m, 256, 0, st>>>(M, (int)K, X, Q, scale);
  else
    quantize_rows_kernel<E><<<m, 256, 0, st>>>(K, X, Q, scale);
  return cudaGetLastError();
}

// ------------------------------------------------------------------ dG and dU
template <int ACT>
__device__ __forceinline__ void gate_backward(float g, float u, float d, float& dg, float& du) {
  const float p = gate_p<ACT>(g);
  dg = d * u * gate_slope<ACT>(g, p);
  du = d * (g * p);
}

// Ten bytes moved for each element and a few dozen instructions: VEC = 8 elements a thread in 128-bit accesses where
// every tensor is 16-byte aligned (8192 x 8192: 105 us, 6.4 TB/s; 174 us one by one).
template <int ACT, bool VEC>
__global__ void __launch_bounds__(256)
gate_backward_kernel(int64_t n, const __nv_bfloat16* G, const __nv_bfloat16* U, const __nv_bfloat16* dH,
                     __nv_bfloat16* dG, __nv_bfloat16* dU) {
  grid_dep_launch();
  const int64_t first = blockIdx.x * (int64_t)256 + threadIdx.x, stride = (int64_t)gridDim.x * 256;
  if (VEC) {
    for (int64_t i = first; i < n / 8; i += stride) {
      float g[8], u[8], d[8];
      widen<__nv_bfloat16>(reinterpret_cast<const uint4*>(G)[i], g);
      widen<__nv_bfloat16>(reinterpret_cast<const uint4*>(U)[i], u);
      widen<__nv_bfloat16>(reinterpret_cast<const uint4*>(dH)[i], d);
      uint32_t wg[4], wu[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float a[2], b[2];
        gate_backward<ACT>(g[2 * j], u[2 * j], d[2 * j], a[0], b[0]);
        gate_backward<ACT>(g[2 * j + 1], u[2 * j + 1], d[2 * j + 1], a[1], b[1]);
        const __nv_bfloat162 x = __floats2bfloat162_rn(a[0], a[1]), y = __floats2bfloat162_rn(b[0], b[1]);
        wg[j] = *reinterpret_cast<const uint32_t*>(&x);
        wu[j] = *reinterpret_cast<const uint32_t*>(&y);
      }
      reinterpret_cast<uint4*>(dG)[i] = make_uint4(wg[0], wg[1], wg[2], wg[3]);
      reinterpret_cast<uint4*>(dU)[i] = make_uint4(wu[0], wu[1], wu[2], wu[3]);
    }
  }
  for (int64_t i = (VEC ? n / 8 * 8 : 0) + first; i < n; i += stride) {
    float dg, du;
    gate_backward<ACT>(__bfloat162float(G[i]), __bfloat162float(U[i]), __bfloat162float(dH[i]), dg, du);
    dG[i] = __float2bfloat16_rn(dg);
    dU[i] = __float2bfloat16_rn(du);
  }
}

template <int ACT>
cudaError_t backward(exo_b200_Context* ctx, int64_t n, const uint16_t* G, const uint16_t* U, const uint16_t* dH,
                     uint16_t* dG, uint16_t* dU) {
  auto r = [](const uint16_t* q) { return reinterpret_cast<const __nv_bfloat16*>(q); };
  auto w = [](uint16_t* q) { return reinterpret_cast<__nv_bfloat16*>(q); };
  const bool vec = aligned16(G) && aligned16(U) && aligned16(dH) && aligned16(dG) && aligned16(dU);
  const int64_t work = vec ? (n + 7) / 8 : n;
  const unsigned grid = (unsigned)std::min<int64_t>((work + 255) / 256, (int64_t)ctx->sm_count * 8);
  if (vec)
    gate_backward_kernel<ACT, true><<<grid, 256, 0, ctx->stream>>>(n, r(G), r(U), r(dH), w(dG), w(dU));
  else
    gate_backward_kernel<ACT, false><<<grid, 256, 0, ctx->stream>>>(n, r(G), r(U), r(dH), w(dG), w(dU));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize_rows(exo_b200_Context* ctx, int64_t M, int64_t K, const void* X, bool bf16, int8_t* Q,
                                 float* scale) {
  return bf16 ? quantize(ctx, M, K, static_cast<const __nv_bfloat16*>(X), Q, scale)
              : quantize(ctx, M, K, static_cast<const float*>(X), Q, scale);
}

cudaError_t launch_gate_backward(exo_b200_Context* ctx, int act, int64_t n, const uint16_t* G, const uint16_t* U,
                                 const uint16_t* dH, uint16_t* dG, uint16_t* dU) {
  return act == EXO_B200_ACT_SILU   ? backward<EXO_B200_ACT_SILU>(ctx, n, G, U, dH, dG, dU)
         : act == EXO_B200_ACT_GELU ? backward<EXO_B200_ACT_GELU>(ctx, n, G, U, dH, dG, dU)
                                    : backward<EXO_B200_ACT_GELU_TANH>(ctx, n, G, U, dH, dG, dU);
}

}  // namespace ffn
}  // namespace exob200
