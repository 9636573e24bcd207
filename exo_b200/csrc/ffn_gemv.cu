// Feed-forward products of at most four rows on the CUDA cores.
//
// With a handful of tokens every weight is multiplied a few times and read once: the time is the weights' way to the
// SMs, and what counts is how soon and how many loads are in flight.  So there is no ring, no tensor memory and no
// cluster to set up: a warp takes R weight rows, reads them 512 bytes at a time with 16-byte loads that bypass L1,
// multiplies against the tokens in shared memory (dp4a, or packed fp32 FMAs of widened bf16), adds over its lanes with
// shuffles, and, where a row is split over KS warps of the CTA, over those through shared memory in a fixed order.
// Rows that do not start on 16 bytes are read by the vectors around them and shifted into place between neighbouring
// lanes, so that no copy is needed.
#include <type_traits>

#include "ffn.cuh"
#include "tc_common.cuh"

namespace exob200 {
namespace ffn {
namespace {

using tc::aligned16;
using umma::grid_dep_launch;
using umma::grid_dep_wait;

constexpr int R = 4;       // weight rows a warp reads at a time (gated: two of the gate, two of the up projection)
constexpr int WARPS = 8;

struct RowArgs {
  int M, N, K;             // tokens, output columns, reduction
  int k_split;             // warps that share a row
  const void *x, *w0, *w1; // tokens (quantised or not), weights
  const float *row_scale, *col_scale, *col_scale1, *bias;
  void *c0, *c1, *c2;
  int8_t* q;               // LINEAR: where CTA 0 leaves the quantised tokens and their scales
  float* q_scale;
  int act;
  int x_vec;               // tokens are whole 16-byte vectors
};

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// v: the aligned vector that holds the first 16 - shift of this lane's 16 bytes, the next lane's the rest (all lanes of
// the warp call this).  Leaves the lane's bytes in v, those from `left` on as zeros.
__device__ __forceinline__ void into_place(uint4& v, uint32_t shift, int left) {
  const uint32_t bits = 8 * (shift & 3u);
  auto next = [](uint32_t w) { return __shfl_down_sync(0xffffffffu, w, 1); };
  auto join = [bits](uint32_t lo, uint32_t hi) { return __funnelshift_r(lo, hi, bits); };
  switch (shift >> 2) {  // the same for the whole warp
    case 0:
      v = make_uint4(join(v.x, v.y), join(v.y, v.z), join(v.z, v.w), join(v.w, next(v.x)));
      break;
    case 1: {
      const uint32_t a = next(v.x), b = next(v.y);
      v = make_uint4(join(v.y, v.z), join(v.z, v.w), join(v.w, a), join(a, b));
      break;
    }
    case 2: {
      const uint32_t a = next(v.x), b = next(v.y), c = next(v.z);
      v = make_uint4(join(v.z, v.w), join(v.w, a), join(a, b), join(b, c));
      break;
    }
    default: {
      const uint32_t a = next(v.x), b = next(v.y), c = next(v.z), d = next(v.w);
      v = make_uint4(join(v.w, a), join(a, b), join(b, c), join(c, d));
    }
  }
  if (left < 16) {
    auto keep = [](uint32_t w, int n) { return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u); };
    v = make_uint4(keep(v.x, left), keep(v.y, left - 4), keep(v.z, left - 8), keep(v.w, left - 12));
  }
}

// ---- multiply-accumulate of one 32-bit word of weights and tokens
template <bool I8>
struct Acc;
template <>
struct Acc<true> {
  int v = 0;
  __device__ __forceinline__ void mac(uint32_t w, uint32_t x) { v = __dp4a((int)w, (int)x, v); }
  __device__ __forceinline__ uint32_t total() const { return (uint32_t)v; }
  static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) { return a + b; }
};
__device__ __forceinline__ uint64_t widen_pair(uint32_t w) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "r"(w << 16), "r"(w & 0xffff0000u));
  return p;
}
template <>
struct Acc<false> {
  uint64_t v = 0;  // two fp32 sums, of the even and the odd elements
  __device__ __forceinline__ void mac(uint64_t w, uint64_t x) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(v) : "l"(w), "l"(x));
  }
  __device__ __forceinline__ uint32_t total() const {
    return __float_as_uint(__uint_as_float((uint32_t)v) + __uint_as_float((uint32_t)(v >> 32)));
  }
  static __device__ __forceinline__ uint32_t add(uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }
};

// v[0 .. V) summed over the warp's lanes; afterwards lane i (i < V) holds the sum of v[i], in v[0].  Each step halves
// the values that a lane carries instead of sending all of them through all five steps.
template <bool I8, int V>
__device__ __forceinline__ uint32_t warp_sums(uint32_t (&v)[V], int lane) {
  int live = V;
#pragma unroll
  for (int bit = 16; bit; bit >>= 1) {
    if (live > 1 && bit < V) {
      live /= 2;
#pragma unroll
      for (int i = 0; i < V / 2; i++) {
        if (i >= live) break;
        const bool upper = lane & bit;
        const uint32_t give = upper ? v[i] : v[i + live], keep = upper ? v[i + live] : v[i];
        v[i] = Acc<I8>::add(keep, __shfl_xor_sync(0xffffffffu, give, bit));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) {
        if (i >= live) break;
        v[i] = Acc<I8>::add(v[i], __shfl_xor_sync(0xffffffffu, v[i], bit));
      }
    }
  }
  return v[0];
}

// Tokens into shared memory, M rows of `pitch` bytes, zeros behind the last element (a whole number of pieces).
__device__ __forceinline__ void load_tokens(const RowArgs& p, uint8_t* s, int pitch, int row_bytes) {
  const uint8_t* x = static_cast<const uint8_t*>(p.x);
  if (p.x_vec) {
    const int per_row = pitch / 16;
    for (int i = threadIdx.x; i < p.M * per_row; i += 32 * WARPS) {
      const int m = i / per_row, c = (i - m * per_row) * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (c < row_bytes) v = *reinterpret_cast<const uint4*>(x + (int64_t)m * row_bytes + c);
      *reinterpret_cast<uint4*>(s + (int64_t)m * pitch + c) = v;
    }
  } else {
    for (int m = 0; m < p.M; m++)
      for (int c = threadIdx.x; c < pitch; c += 32 * WARPS)
        s[m * pitch + c] = c < row_bytes ? x[(int64_t)m * row_bytes + c] : 0;
  }
}

// The same for tokens that are quantised on the way; every CTA does so for itself, CTA 0 also writes them out.
// scale[m] is left in shared memory.
template <class XT, int MR>
__device__ __forceinline__ void quantize_tokens(const RowArgs& p, uint8_t* s, int pitch, float* scale) {
  constexpr int N = 16 / sizeof(XT);
  __shared__ unsigned tops[MR][WARPS];
  const XT* x = static_cast<const XT*>(p.x);
  unsigned top[MR] = {};
#pragma unroll
  for (int m = 0; m < MR; m++) {
    if (m >= p.M) break;
    const XT* row = x + (int64_t)m * p.K;
    if (p.x_vec) {
      for (int k = threadIdx.x * N; k < p.K; k += 32 * WARPS * N) {
        float f[N];
        widen<XT>(*reinterpret_cast<const uint4*>(row + k), f);
#pragma unroll
        for (int j = 0; j < N; j++) top[m] = max(top[m], magnitude(f[j]));
      }
    } else {
      for (int k = threadIdx.x; k < p.K; k += 32 * WARPS) top[m] = max(top[m], magnitude(float(row[k])));
    }
    top[m] = __reduce_max_sync(0xffffffffu, top[m]);
    if (threadIdx.x % 32 == 0) tops[m][threadIdx.x / 32] = top[m];
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MR; m++) {
    if (m >= p.M) break;
#pragma unroll
    for (int w = 0; w < WARPS; w++) top[m] = max(top[m], tops[m][w]);
    const Step step = step_of(top[m]);
    if (threadIdx.x == 0) {
      scale[m] = step.scale;
      if (blockIdx.x == 0) p.q_scale[m] = step.scale;
    }
    const XT* row = x + (int64_t)m * p.K;
    if (p.x_vec) {
      for (int k = threadIdx.x * N; k < pitch; k += 32 * WARPS * N) {
        uint32_t w[N / 4] = {};
        if (k < p.K) {
          float f[N];
          widen<XT>(*reinterpret_cast<const uint4*>(row + k), f);
#pragma unroll
          for (int j = 0; j < N; j++) w[j / 4] |= quantized(f[j], step) << (8 * (j % 4));
        }
#pragma unroll
        for (int j = 0; j < N / 4; j++) {
          *reinterpret_cast<uint32_t*>(s + m * pitch + k + 4 * j) = w[j];
          if (blockIdx.x == 0 && k < p.K) *reinterpret_cast<uint32_t*>(p.q + (int64_t)m * p.K + k + 4 * j) = w[j];
        }
      }
    } else {
      for (int k = threadIdx.x; k < pitch; k += 32 * WARPS) {
        const uint8_t v = k < p.K ? (uint8_t)quantized(float(row[k]), step) : 0;
        s[m * pitch + k] = v;
        if (blockIdx.x == 0 && k < p.K) p.q[(int64_t)m * p.K + k] = (int8_t)v;
      }
    }
  }
}

// Pieces of each row in flight in a warp.
template <bool I8, int MR, bool VEC>
__host__ __device__ constexpr int batch() {
  // measured: bf16 1 x 16384 x 4096 gated 43.5 us with four, 44.7 with two; int8 21.8 with two, 22.7 with four;
  // unaligned rows want registers more than loads in flight (K = 4095: 55.3 us with one, 66.6 with two)
  return !VEC ? 1 : !I8 && MR <= 2 ? 4 : 2;
}

// XT: what the tokens are quantised from (void: they come as the product takes them).
template <int KIND, class O, int MR, bool VEC, class XT>
__global__ void __launch_bounds__(32 * WARPS)
row_kernel(const __grid_constant__ RowArgs p) {
  constexpr bool I8 = KIND != GATED, TWO = KIND != SCALED;
  constexpr int E = I8 ? 1 : 2;
  constexpr int V = R * MR;
  constexpr int COLS = TWO ? R / 2 : R;  // output columns of a group
  // bytes of a row that a warp takes at a time; unaligned rows give lane 31's vector to lane 30
  constexpr int PIECE = VEC ? 512 : 496;
  constexpr int BATCH = batch<I8, MR, VEC>();
  extern __shared__ __align__(16) uint8_t tokens[];
  __shared__ uint32_t sums[2][WARPS][V];
  __shared__ float token_scale[MR];
  constexpr bool LINEAR = !std::is_void<XT>::value;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_bytes = p.K * E, pitch = (row_bytes + 511) / 512 * 512;
  const int pieces = (row_bytes + PIECE - 1) / PIECE;
  const int groups = (p.N + COLS - 1) / COLS, per_cta = WARPS / p.k_split;
  const int ks = warp % p.k_split, slot = warp / p.k_split;

  grid_dep_wait();
  if constexpr (LINEAR)
    quantize_tokens<XT, MR>(p, tokens, pitch, token_scale);
  else
    load_tokens(p, tokens, pitch, row_bytes);
  __syncthreads();

  int buffer = 0;
  for (int base = blockIdx.x * per_cta; base < groups; base += gridDim.x * per_cta, buffer ^= 1) {
    const int group = base + slot;
    const int col0 = group * COLS;
    Acc<I8> acc[R][MR];
    if (group < groups) {
      const uint8_t* row[R];
      uint32_t shift[R];  // bytes of the first 16-byte vector in front of the row
#pragma unroll
      for (int r = 0; r < R; r++) {
        // rows past the last are read again in its place; their sums are not stored
        const int n = min(col0 + (TWO ? r % COLS : r), p.N - 1);
        row[r] = static_cast<const uint8_t*>(TWO && r >= COLS ? p.w1 : p.w0) + (int64_t)n * row_bytes;
        shift[r] = VEC ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(row[r]) & 15u);
        row[r] -= shift[r];
      }
      for (int piece = ks; piece < pieces; piece += p.k_split * BATCH) {
        uint4 w[BATCH][R];
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
          const int at = (piece + b * p.k_split) * PIECE + lane * 16;
#pragma unroll
          for (int r = 0; r < R; r++)  // vectors that hold a byte of the row
            w[b][r] = at < row_bytes + (int)shift[r] ? ld_stream(row[r] + at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
          const int at = (piece + b * p.k_split) * PIECE + lane * 16;
          if (!VEC) {
#pragma unroll
            for (int r = 0; r < R; r++) into_place(w[b][r], shift[r], row_bytes - at);
            if (lane == 31) continue;  // its vector was the other half of lane 30's
          }
          if (at >= pitch) continue;
#pragma unroll
          for (int m = 0; m < MR; m++) {
            if (MR > 1 && m >= p.M) break;
            const uint4 x = *reinterpret_cast<const uint4*>(tokens + m * pitch + at);
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int r = 0; r < R; r++) {
              const uint32_t ws[4] = {w[b][r].x, w[b][r].y, w[b][r].z, w[b][r].w};
#pragma unroll
              for (int j = 0; j < 4; j++) {
                if constexpr (I8)
                  acc[r][m].mac(ws[j], xs[j]);
                else
                  acc[r][m].mac(widen_pair(ws[j]), widen_pair(xs[j]));
              }
            }
          }
        }
      }
    }
    uint32_t v[V];
#pragma unroll
    for (int m = 0; m < MR; m++)
#pragma unroll
      for (int r = 0; r < R; r++) v[m * R + r] = acc[r][m].total();
    const uint32_t mine = warp_sums<I8, V>(v, lane);
    if (lane < V) sums[buffer][warp][lane] = mine;
    if (p.k_split > 1)
      __syncthreads();
    else
      __syncwarp();
    if (ks == 0 && group < groups && lane < MR * COLS) {
      const int m = lane / COLS, c = lane % COLS, col = col0 + c;
      if (m < p.M && col < p.N) {
        auto sum = [&](int r) {
          uint32_t s = sums[buffer][warp][m * R + r];
          for (int k = 1; k < p.k_split; k++) s = Acc<I8>::add(s, sums[buffer][warp + k][m * R + r]);
          return s;
        };
        const int64_t at = (int64_t)m * p.N + col;
        if constexpr (KIND == SCALED) {
          const float y = scaled((int32_t)sum(c), LINEAR ? token_scale[m] : p.row_scale[m], __ldg(p.col_scale + col)) +
                          (p.bias ? __ldg(p.bias + col) : 0.f);
          static_cast<O*>(p.c0)[at] = O(y);
        } else {
          float g, u;
          if constexpr (I8) {
            const float rs = p.row_scale[m];
            g = scaled((int32_t)sum(c), rs, __ldg(p.col_scale + col));
            u = scaled((int32_t)sum(COLS + c), rs, __ldg(p.col_scale1 + col));
          } else {
            g = __uint_as_float(sum(c));
            u = __uint_as_float(sum(COLS + c));
          }
          const float a = p.act == EXO_B200_ACT_SILU   ? gate<EXO_B200_ACT_SILU>(g)
                          : p.act == EXO_B200_ACT_GELU ? gate<EXO_B200_ACT_GELU>(g)
                                                       : gate<EXO_B200_ACT_GELU_TANH>(g);
          static_cast<O*>(p.c0)[at] = O(a * u);
          if (p.c1) {
            static_cast<O*>(p.c1)[at] = O(g);
            static_cast<O*>(p.c2)[at] = O(u);
          }
        }
      }
    }
  }
}

template <int KIND, class O, int MR, bool VEC, class XT>
cudaError_t go(exo_b200_Context* ctx, const RowArgs& a, int grid, size_t smem, bool after_own_kernel) {
  auto* kernel = row_kernel<KIND, O, MR, VEC, XT>;
  EXOB200_SMEM_ATTR_ONCE(kernel, kRowTokenBytes, ctx->device);
  if (after_own_kernel) return tc::launch_dependent(kernel, dim3(grid), dim3(32 * WARPS), smem, ctx->stream, a);
  kernel<<<grid, 32 * WARPS, smem, ctx->stream>>>(a);
  return cudaGetLastError();
}

template <int KIND, class O, class XT = void>
cudaError_t launch(exo_b200_Context* ctx, const Problem& p, bool after_own_kernel, const void* X = nullptr) {
  constexpr int E = KIND == GATED ? 2 : 1, COLS = KIND == SCALED ? R : R / 2;
  RowArgs a{};
  a.M = (int)p.M, a.N = (int)p.N, a.K = (int)p.K;
  a.x = p.a0, a.w0 = p.b0, a.w1 = p.b1;
  a.row_scale = p.row_scale, a.col_scale = p.col_scale, a.col_scale1 = p.col_scale1, a.bias = p.bias;
  a.c0 = p.c0, a.c1 = p.c1, a.c2 = p.c2;
  a.act = p.act;
  const int64_t row_bytes = p.K * E;
  if (X) {
    a.x = X;
    a.q = static_cast<int8_t*>(const_cast<void*>(p.a0));
    a.q_scale = const_cast<float*>(p.row_scale);
    constexpr int N = std::is_same<XT, float>::value ? 4 : 8;  // elements of a vector of X
    a.x_vec = p.K % N == 0 && aligned16(X) && reinterpret_cast<uintptr_t>(a.q) % 4 == 0;
  } else {
    a.x_vec = row_bytes % 16 == 0 && aligned16(p.a0);
  }
  const bool vec = row_bytes % 16 == 0 && aligned16(p.b0) && (KIND == SCALED || aligned16(p.b1));
  const int64_t groups = (p.N + COLS - 1) / COLS;
  // Eight warps an SM, or 24 that have one piece in flight, keep the memory busy: split rows over the CTA's warps while
  // there are fewer.
  a.k_split = 1;
  const int64_t piece = vec ? 512 : 496, pieces = (row_bytes + piece - 1) / piece;
  while (a.k_split < WARPS && groups * a.k_split < (vec ? 8 : 24) * ctx->sm_count && pieces >= 2 * a.k_split) a.k_split *= 2;
  const int64_t ctas = (groups * a.k_split + WARPS - 1) / WARPS;
  const size_t smem = (size_t)(p.M * ((row_bytes + 511) / 512 * 512));
  const int per_sm = smem <= 32768 ? 4 : 2;
  const int grid = (int)std::min<int64_t>(ctas, (int64_t)per_sm * ctx->sm_count);
  const int mr = p.M <= 1 ? 1 : p.M <= 2 ? 2 : 4;
  const bool own = after_own_kernel;
  if (vec)
    return mr == 1   ? go<KIND, O, 1, true, XT>(ctx, a, grid, smem, own)
           : mr == 2 ? go<KIND, O, 2, true, XT>(ctx, a, grid, smem, own)
                     : go<KIND, O, 4, true, XT>(ctx, a, grid, smem, own);
  return mr == 1   ? go<KIND, O, 1, false, XT>(ctx, a, grid, smem, own)
         : mr == 2 ? go<KIND, O, 2, false, XT>(ctx, a, grid, smem, own)
                   : go<KIND, O, 4, false, XT>(ctx, a, grid, smem, own);
}

}  // namespace

bool rows_wanted(Kind kind, const Problem& p) {
  static const int mode = [] {
    const char* e = getenv("EXOB200_FFN_ROWS");
    return e ? atoi(e) : -1;
  }();
  const int64_t pitch = (p.K * (kind == GATED ? 2 : 1) + 511) / 512 * 512;
  if (mode == 0 || kind == DGRAD || kind == WGRAD || p.M > 4) return false;
  if (p.M * pitch > kRowTokenBytes) return false;
  // From three bf16 tokens on the arithmetic outlasts the weights' way here: the tensor cores take large problems
  // (4 x 16384 x 4096 gated: 56.3 us here, 48.4 there; 4 x 4099 x 513: 9.8 and 11.3)
  return kind != GATED || p.M <= 2 || p.N * p.K <= (int64_t)8 << 20;
}

// Every CTA quantises all tokens, so they have to be few (1 x 4096 tokens for 4096 channels: 6.1 us in one kernel, 6.6 in
// two; 4 x 4096: 9.9 and 8.7), though each launch also costs the host 2 us.
bool linear_rows_wanted(const Problem& p, bool f32) {
  return rows_wanted(SCALED, p) && p.M * p.K * (f32 ? 4 : 2) <= 16384;
}

cudaError_t launch_linear_rows(exo_b200_Context* ctx, bool f32, const Problem& p, const void* X) {
  return f32 ? launch<SCALED, float, float>(ctx, p, false, X)
             : launch<SCALED, __nv_bfloat16, __nv_bfloat16>(ctx, p, false, X);
}

cudaError_t launch_rows(exo_b200_Context* ctx, Kind kind, bool out_f32, const Problem& p, bool after_own_kernel) {
  switch (kind) {
    case SCALED:
      return out_f32 ? launch<SCALED, float>(ctx, p, after_own_kernel)
                     : launch<SCALED, __nv_bfloat16>(ctx, p, after_own_kernel);
    case GATED:
      return launch<GATED, __nv_bfloat16>(ctx, p, after_own_kernel);
    default:
      return launch<GATED_I8, __nv_bfloat16>(ctx, p, after_own_kernel);
  }
}

}  // namespace ffn
}  // namespace exob200
