// Feed-forward products on the tensor cores.
//
// split_kernel: one 128 x 128 accumulator per CTA (gated: 64 columns of the gate and the same 64 of the up projection
// side by side, so that one thread of the epilogue meets both).  TMA -> mbarrier ring -> tcgen05.mma -> tensor memory,
// as in tc_gemm.cu; the reduction is split over the CTAs of a cluster, which add their accumulators through
// distributed shared memory in a fixed order, so results do not depend on timing.
//
// pair_kernel: 256 x 256 tiles on CTA pairs (cta_group::2), persistent, for problems with enough of them.  The pair's
// B tile is half in each CTA's shared memory: for the gated kinds the even CTA loads 128 rows of the gate's weight and
// the odd one the same 128 rows of the up projection's, and every accumulator row holds both.  Where there are few tiles
// and a long reduction, the pairs of a cluster split it as the split kernel's CTAs do.
//
// tall_kernel: 512 x 256 tiles on CTA pairs for the largest problems with one weight.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>

#include "ffn.cuh"
#include "tc_common.cuh"
#include "umma.cuh"
#include "umma_pair.cuh"

namespace exob200 {
namespace ffn {
namespace {

using namespace tc;
using namespace umma;

template <int KIND>
struct Traits {
  static constexpr bool I8 = KIND == SCALED || KIND == GATED_I8;
  static constexpr bool TWO = KIND == GATED || KIND == GATED_I8;  // two weights, two accumulators side by side
  static constexpr bool A_MN = KIND == WGRAD;                     // the reduction runs down A's rows
  static constexpr bool B_MN = KIND == WGRAD || KIND == DGRAD;
  static constexpr int ELEM = I8 ? 1 : 2;
  static constexpr int BK = ROW_BYTES / ELEM;  // reduction elements of a stage
  static constexpr int MMA = I8 ? KIND_I8 : KIND_F16;
  __host__ __device__ static constexpr uint32_t idesc(uint32_t m, uint32_t n) {
    return make_idesc(I8 ? 2 : 1, 1, 1, m, n) | (A_MN ? 1u << 15 : 0u) | (B_MN ? IDESC_B_MN_MAJOR : 0u);
  }
  // descriptor step of one MMA (32 bytes of the reduction) in units of 16 bytes
  __host__ __device__ static constexpr uint64_t step(bool mn) { return mn ? (uint64_t)((32 / ELEM) * ROW_BYTES / 16) : 2u; }
};

struct Args {
  int M, N;              // an output's rows and columns
  int nkb, segments;     // k-blocks of one operand pair; DGRAD runs over two
  int tiles_m, tiles_n;
  int a_rows;            // rows of A's box (fewer than 128 when M is)
  int vec;               // outputs take vector stores
  int b_early;           // the kernel before this one may still run, and writes neither B nor the scales of its columns
  int let_beside;        // successors may start once this kernel has what it waits for
  int wait_last;         // beside the kernel before it: waits for that one only before it ends
  const float *row_scale, *col_scale, *col_scale1, *bias;
  void *c0, *c1, *c2;
  DeviceStatus* status;
  const uint8_t *a, *b, *b1;  // operands that are gathered instead of copied by TMA; rows of row_bytes
  int row_bytes;
};

// What the kernel before this one wrote may be read from here on.
__device__ __forceinline__ void wait_before(const Args& p) {
  if (!p.wait_last) grid_dep_wait();
  if (p.let_beside) grid_dep_launch();
}

// ------------------------------------------------------------------ epilogue arithmetic
template <class O>
__device__ __forceinline__ void store4(O* p, const float (&v)[4], int left, bool vec);
template <>
__device__ __forceinline__ void store4<float>(float* p, const float (&v)[4], int left, bool vec) {
  if (vec && left >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < left) p[j] = v[j];
  }
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[4], int left, bool vec) {
  if (vec && left >= 4) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < left) p[j] = __float2bfloat16_rn(v[j]);
  }
}

// What a thread needs of four neighbouring output columns for any number of rows.
template <int KIND>
struct Columns {
  using T = Traits<KIND>;
  int col, left;
  float scale[T::I8 ? 4 : 1], scale1[T::I8 && T::TWO ? 4 : 1], bias[KIND == SCALED ? 4 : 1];

  __device__ __forceinline__ Columns(const Args& p, int c) : col(c), left(p.N - c) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const bool in = j < left;
      if constexpr (T::I8) scale[j] = in ? __ldg(p.col_scale + col + j) : 0.f;
      if constexpr (T::I8 && T::TWO) scale1[j] = in ? __ldg(p.col_scale1 + col + j) : 0.f;
      if constexpr (KIND == SCALED) bias[j] = in && p.bias ? __ldg(p.bias + col + j) : 0.f;
    }
  }
};

// Those columns of one output row, from finished sums.
template <int KIND, class O, int ACT>
__device__ __forceinline__ void finish4(const Args& p, const Columns<KIND>& k, int z, int row, float rs,
                                        const uint32_t (&x)[4], const uint32_t (&y)[4]) {
  using T = Traits<KIND>;
  const int64_t at = (int64_t)row * p.N + k.col;
  float v[4], g[4], u[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if constexpr (KIND == SCALED) {
      v[j] = scaled((int32_t)x[j], rs, k.scale[j]) + k.bias[j];
    } else if constexpr (KIND == GATED_I8) {
      g[j] = scaled((int32_t)x[j], rs, k.scale[j]);
      u[j] = scaled((int32_t)y[j], rs, k.scale1[j]);
    } else {
      v[j] = g[j] = __uint_as_float(x[j]);
      u[j] = __uint_as_float(y[j]);
    }
    if constexpr (T::TWO) v[j] = gate<ACT>(g[j]) * u[j];
  }
  if (T::TWO && p.c1) {
    store4(static_cast<O*>(p.c1) + at, g, k.left, p.vec);
    store4(static_cast<O*>(p.c2) + at, u, k.left, p.vec);
  }
  store4(static_cast<O*>(KIND == WGRAD && z ? p.c1 : p.c0) + at, v, k.left, p.vec);
}

// ------------------------------------------------------------------ split kernel
// A stage is 128 rows of B and as many of A as there are (in eights); the ring is as deep as its share of the SM takes:
// all of it where the grid leaves an SM to each CTA, half of it otherwise.  The loads in flight are what counts: a
// CTA alone on its SM with three stages of 32 KiB took 0.47 us a k-block, waiting for L2, 0.43 with six.
constexpr int S_MAX_STAGES = 12;
constexpr int S_CTRL = 1024 + 256;                 // alignment, barriers
constexpr int S_SMEM_ALONE = 232448, S_SMEM_SHARED = 233472 / 2 - 1024;
constexpr int S_PITCH = 132;                       // words between rows of the accumulator in shared memory: 128-bit
                                                   // accesses of neighbouring rows fall on different banks
// the accumulator takes the ring's place
static_assert(BM * S_PITCH * 4 <= (S_SMEM_SHARED - S_CTRL) / (2 * A_TILE_BYTES) * (2 * A_TILE_BYTES), "");
constexpr uint32_t S_TMEM_COLS = 128;
constexpr int MAX_SPLIT = 16;  // CTAs of a cluster; above eight the size is not portable, but this GPU takes it

__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
template <bool I8>
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) {
  return I8 ? a + b : __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}
// Sum over S CTAs of the cluster, of ranks first, first + RANKS, ..., of the four accumulator words at `offset`; always
// in the order of the ranks.
template <bool I8, int S, int RANKS>
__device__ __forceinline__ void cluster_sum(uint32_t base, uint32_t offset, int first, uint32_t (&x)[4]) {
  uint4 v[S];
#pragma unroll
  for (int s = 0; s < S; s++) v[s] = ld_cluster_v4(mapa(base, (uint32_t)(first + s * RANKS)) + offset);
  x[0] = v[0].x, x[1] = v[0].y, x[2] = v[0].z, x[3] = v[0].w;
#pragma unroll
  for (int s = 1; s < S; s++) {
    x[0] = plus<I8>(x[0], v[s].x);
    x[1] = plus<I8>(x[1], v[s].y);
    x[2] = plus<I8>(x[2], v[s].z);
    x[3] = plus<I8>(x[3], v[s].w);
  }
}

// Rows split, split + S, ... of a CTA's 128 (from m0): sums over the cluster, epilogue, stores.  The accumulators lie in
// shared memory, COLS columns in rows of PITCH words.  A thread keeps its four columns and goes down the rows, several
// at a time so that their round trips overlap.
template <int KIND, class O, int ACT, int THREADS, int S, int COLS, int PITCH, int RANKS>
__device__ __forceinline__ void cluster_epilogue(const Args& p, uint32_t base, int split, int first_rank, int z, int m0,
                                                 int n0) {
  using T = Traits<KIND>;
  constexpr int GROUPS = (T::TWO ? COLS / 2 : COLS) / 4;  // groups of four output columns
  constexpr int STEP = THREADS / GROUPS;                  // rows that the CTA covers at a time
  constexpr int BATCH = S > 4 ? 1 : S > 2 ? 2 : 4;
  static_assert(THREADS % GROUPS == 0, "a thread keeps its columns");
  const Columns<KIND> cols(p, n0 + (int)threadIdx.x % GROUPS * 4);
  if (cols.left <= 0) return;
  const int rows = (min(BM, p.M - m0) - split + S - 1) / S;
  const uint32_t c = (uint32_t)threadIdx.x % GROUPS * 16u;
  for (int first = threadIdx.x / GROUPS; first < rows; first += STEP * BATCH) {
    uint32_t x[BATCH][4], y[BATCH][4] = {};
    float rs[BATCH] = {};
#pragma unroll
    for (int b = 0; b < BATCH; b++) {
      const int r = split + min(first + b * STEP, rows - 1) * S;
      if constexpr (T::I8) rs[b] = p.row_scale[m0 + r];
      const uint32_t at = (uint32_t)(r * PITCH) * 4u + c;
      cluster_sum<T::I8, S, RANKS>(base, at, first_rank, x[b]);
      if constexpr (T::TWO) cluster_sum<T::I8, S, RANKS>(base, at + COLS / 2 * 4, first_rank, y[b]);
    }
#pragma unroll
    for (int b = 0; b < BATCH; b++)
      if (first + b * STEP < rows)
        finish4<KIND, O, ACT>(p, cols, z, m0 + split + (first + b * STEP) * S, rs[b], x[b], y[b]);
  }
}

// ---- gathered operands
// Rows whose pitch or base TMA cannot take are read by the aligned 16-byte vectors around them (nine for 128 bytes),
// asynchronously into a ring of raw rows in shared memory, and shifted from there into the swizzled tile.  A warp
// shifts what it has fetched itself, so no two warps wait for one another.
constexpr int G_WARPS = 8;                      // warps 2 .. 9 gather
constexpr int G_THREADS = 64 + 32 * G_WARPS;
constexpr int G_STAGES = 2;                     // swizzled tiles
constexpr int G_RAW_ROW = ROW_BYTES + 16;
constexpr int G_MAX_M = 32;                     // tokens: with more, shifting takes longer than copies do
constexpr int G_DEPTH = 3;                      // raw k-blocks, two of them in flight while one is shifted
constexpr int G_A_TILE = G_MAX_M * ROW_BYTES, G_STAGE_BYTES = G_A_TILE + A_TILE_BYTES;
constexpr int G_RAW = (G_MAX_M + BM) * G_RAW_ROW;
constexpr int G_AREA = G_STAGES * G_STAGE_BYTES + G_DEPTH * G_RAW;
constexpr int G_SMEM = G_AREA + S_CTRL;
static_assert(G_AREA >= BM * S_PITCH * 4, "the accumulator takes the rings' place");
static_assert(G_SMEM <= S_SMEM_SHARED, "two CTAs share an SM");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
  const int bytes = in ? 16 : 0;  // zeros otherwise
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Sixteen bytes that start `shift` bytes into the aligned vector lo and end in the next one, hi.  Selects, no branches:
// the shift differs between the rows of a warp.
__device__ __forceinline__ uint4 join16(const uint4& lo, const uint4& hi, uint32_t shift) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  const bool two = shift & 8u, one = shift & 4u;
#pragma unroll
  for (int j = 0; j < 6; j++) w[j] = two ? w[j + 2] : w[j];
#pragma unroll
  for (int j = 0; j < 5; j++) w[j] = one ? w[j + 1] : w[j];
  const uint32_t bits = 8 * (shift & 3u);
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// One row of an operand as eight lanes share it.
struct GatherRow {
  const uint8_t* aligned;  // the row's first vector; nullptr: no such row
  uint32_t shift;          // bytes of it in front of the row

  __device__ __forceinline__ void set(const uint8_t* row) {
    shift = (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u);
    aligned = row ? row - shift : nullptr;
  }
  // vectors [at, at + 144) of the row, those that hold none of its bytes as zeros
  __device__ __forceinline__ void fetch(uint32_t raw, int at, int row_bytes, int v) const {
    if (!aligned) return;
    const int end = row_bytes + (int)shift;
    cp_async16(raw + v * 16, at + v * 16 < end ? aligned + at + v * 16 : aligned, at + v * 16 < end);
    if (v == 7) cp_async16(raw + 128, at + 128 < end ? aligned + at + 128 : aligned, at + 128 < end);
  }
  // bytes [at + 16 v, + 16) of the row to their swizzled place in line r of a tile
  __device__ __forceinline__ void place(uint32_t raw, uint32_t tile, int r, int at, int row_bytes, int v) const {
    if (!aligned) return;
    const uint4 joined = join16(ld_shared16(raw + v * 16), ld_shared16(raw + v * 16 + 16), shift);
    uint32_t y[4] = {joined.x, joined.y, joined.z, joined.w};
    const int left = row_bytes - at - v * 16;
    if (left < 16) {  // nothing behind the row's end may reach a sum
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int keep = left - 4 * j;
        if (keep < 4) y[j] = keep <= 0 ? 0u : y[j] & ((1u << (8 * keep)) - 1u);
      }
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(tile + (uint32_t)(r * ROW_BYTES + ((v ^ (r & 7)) * 16))),
                 "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3])
                 : "memory");
  }
};

// The gathering warps' part of a CTA: warp w takes rows 4 (w + 8 i) + lane / 8 of the B tile and of A.
template <int KIND>
__device__ __forceinline__ void gather(const Args& p, uint32_t tiles, uint32_t full0, uint32_t empty0,
                                       volatile int* abort_flag, int w, int lane, int m0, int n0, int kb0, int n_kb) {
  using T = Traits<KIND>;
  constexpr int B_ROWS = BM / (4 * G_WARPS);
  const uint32_t raw0 = tiles + G_STAGES * G_STAGE_BYTES;
  const int v = lane & 7, first = w * 4 + lane / 8;
  GatherRow a, b[B_ROWS];
  a.set(m0 + first < p.M ? p.a + (int64_t)(m0 + first) * p.row_bytes : nullptr);
#pragma unroll
  for (int i = 0; i < B_ROWS; i++) {
    const int r = first + 32 * i, n = n0 + (T::TWO ? r % 64 : r);
    b[i].set(n < p.N ? (T::TWO && r >= 64 ? p.b1 : p.b) + (int64_t)n * p.row_bytes : nullptr);
  }
  auto fetch = [&](int i) {
    if (i < n_kb) {
      const uint32_t raw = raw0 + (uint32_t)(i % G_DEPTH * G_RAW);
      const int at = (kb0 + i) * ROW_BYTES;
      a.fetch(raw + first * G_RAW_ROW, at, p.row_bytes, v);
#pragma unroll
      for (int j = 0; j < B_ROWS; j++)
        b[j].fetch(raw + (G_MAX_M + first + 32 * j) * G_RAW_ROW, at, p.row_bytes, v);
    }
    cp_async_commit();  // a group for every k-block, empty ones behind the last
  };
#pragma unroll
  for (int i = 0; i < G_DEPTH - 1; i++) fetch(i);
  int stage = 0;
  uint32_t phase = 1;
  for (int i = 0; i < n_kb; i++) {
    fetch(i + G_DEPTH - 1);  // into the slot that this warp has read in the last round
    cp_async_wait<G_DEPTH - 1>();
    __syncwarp();  // the wait shows a lane its own copies, and place() reads its neighbour's, too
    // the lanes decide together, so that none is left alone at a barrier
    if (!__all_sync(0xffffffffu, mbar_wait(empty0 + 8u * stage, phase, abort_flag, WAIT_LIMIT_NS))) {
      if (lane == 0) report_timeout(p.status, abort_flag, 64);
      break;
    }
    const uint32_t raw = raw0 + (uint32_t)(i % G_DEPTH * G_RAW), a_dst = tiles + stage * G_STAGE_BYTES;
    const int at = (kb0 + i) * ROW_BYTES;
    a.place(raw + first * G_RAW_ROW, a_dst, first, at, p.row_bytes, v);
#pragma unroll
    for (int j = 0; j < B_ROWS; j++)
      b[j].place(raw + (G_MAX_M + first + 32 * j) * G_RAW_ROW, a_dst + G_A_TILE, first + 32 * j, at, p.row_bytes, v);
    fence_proxy_async();  // the tensor core reads what was stored here
    __syncwarp();
    if (lane == 0) mbar_arrive(full0 + 8u * stage);
    if (++stage == G_STAGES) {
      stage = 0;
      phase ^= 1u;
    }
  }
  cp_async_wait<0>();
}

template <int KIND, class O, int ACT, bool GATHER>
__global__ void __launch_bounds__(GATHER ? G_THREADS : NUM_THREADS, 2)
split_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmA1,
             const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1,
             const __grid_constant__ Args p, int S, int ring_stages) {
  using T = Traits<KIND>;
  constexpr int BK = T::BK;
  constexpr int CN = T::TWO ? 64 : 128;  // output columns of a tile
  constexpr int THREADS = GATHER ? G_THREADS : NUM_THREADS;
  constexpr uint32_t IDESC = T::idesc(BM, 128);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const int stages = GATHER ? G_STAGES : ring_stages;
  // The MMA reads 128 rows of A whatever there are: those behind a_rows are B's bytes, and their sums are not stored.
  const int a_tile = GATHER ? G_A_TILE : T::A_MN ? A_TILE_BYTES : p.a_rows * ROW_BYTES;
  const int stage_bytes = a_tile + A_TILE_BYTES;
  const uint32_t bars = tiles + (GATHER ? G_AREA : stages * stage_bytes);
  uint8_t* ctrl = smem_raw + (bars - raw);
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (S_MAX_STAGES + s); };
  const uint32_t done_bar = bars + 8u * (2 * S_MAX_STAGES);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl + 8 * (2 * S_MAX_STAGES + 1));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 8 * (2 * S_MAX_STAGES + 1) + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)blockIdx.x % S;  // the cluster is S consecutive CTAs
  int t = (int)blockIdx.x / S;
  const int per_z = p.tiles_m * p.tiles_n;
  const int z = t / per_z;
  t -= z * per_z;
  const int m0 = t % p.tiles_m * BM, n0 = t / p.tiles_m * CN;
  const int total = p.nkb * p.segments;
  const int kb0 = (int)((int64_t)total * rank / S), n_kb = (int)((int64_t)total * (rank + 1) / S) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; s++) {
      mbar_init(full_bar(s), GATHER ? G_WARPS : 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (!GATHER && warp == 2 && lane == 0) {  // the descriptors' first fetch overlaps the set-up
    prefetch_tensormap(&tmA0);
    prefetch_tensormap(&tmB0);
    if (KIND == WGRAD || KIND == DGRAD) prefetch_tensormap(&tmA1);
    if (T::TWO || KIND == DGRAD) prefetch_tensormap(&tmB1);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), S_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (!GATHER && lane == 0) {
      const uint32_t a_bytes = (uint32_t)a_tile;
      auto load_a = [&](int s, int kb) {
        const bool second = kb >= p.nkb;
        const int k0 = (second ? kb - p.nkb : kb) * BK;
        const CUtensorMap* m = second || (KIND == WGRAD && z) ? &tmA1 : &tmA0;
        const uint32_t dst = tiles + s * stage_bytes;
        if (T::A_MN) {
          for (int c = 0; c < 2; c++) tma_load_2d(dst + c * (A_TILE_BYTES / 2), m, full_bar(s), m0 + 64 * c, k0);
        } else {
          tma_load_2d(dst, m, full_bar(s), k0, m0);
        }
      };
      auto load_b = [&](int s, int kb) {
        const bool second = kb >= p.nkb;
        const int k0 = (second ? kb - p.nkb : kb) * BK;
        const uint32_t dst = tiles + s * stage_bytes + a_tile;
        if (T::TWO) {
          tma_load_2d(dst, &tmB0, full_bar(s), k0, n0);
          tma_load_2d(dst + A_TILE_BYTES / 2, &tmB1, full_bar(s), k0, n0);
        } else if (T::B_MN) {
          const CUtensorMap* m = second ? &tmB1 : &tmB0;
          for (int c = 0; c < 2; c++) tma_load_2d(dst + c * (A_TILE_BYTES / 2), m, full_bar(s), n0 + 64 * c, k0);
        } else {
          tma_load_2d(dst, &tmB0, full_bar(s), k0, n0);
        }
      };
      // The ring's first fill.  Beside a kernel of this call, what that kernel does not write comes before waiting for
      // it; otherwise stage by stage, as the MMAs want it.
      const int first = min(n_kb, stages);
      if (p.b_early) {
        for (int i = 0; i < first; i++) {
          mbar_arrive_expect_tx(full_bar(i), a_bytes + A_TILE_BYTES);
          load_b(i, kb0 + i);
        }
        wait_before(p);
        for (int i = 0; i < first; i++) load_a(i, kb0 + i);
      } else {
        wait_before(p);
        for (int i = 0; i < first; i++) {
          mbar_arrive_expect_tx(full_bar(i), a_bytes + A_TILE_BYTES);
          load_b(i, kb0 + i);
          load_a(i, kb0 + i);
        }
      }
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = first; i < n_kb; i++) {
        if (!mbar_wait(empty_bar(stage), phase, abort_flag, WAIT_LIMIT_NS)) {
          report_timeout(p.status, abort_flag, 61);
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(full_bar(stage), a_bytes + A_TILE_BYTES);
        load_b(stage, kb0 + i);
        load_a(stage, kb0 + i);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok || *abort_flag) {  // error path: copies in flight land before the CTA leaves
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < n_kb; i++) {
        if (!mbar_wait(full_bar(stage), phase, abort_flag, WAIT_LIMIT_NS)) {
          report_timeout(p.status, abort_flag, 62);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a0 = tiles + stage * stage_bytes, b0 = a0 + a_tile;
        const uint64_t da = T::A_MN ? smem_desc_mn_sw128(a0, BK) : smem_desc_k_sw128(a0);
        const uint64_t db = T::B_MN ? smem_desc_mn_sw128(b0, BK) : smem_desc_k_sw128(b0);
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++)
          tc_mma<T::MMA>(tmem, da + ks * T::step(T::A_MN), db + ks * T::step(T::B_MN), IDESC, (i | ks) != 0);
        tc_commit(empty_bar(stage));
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) tc_commit(done_bar);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;  // a warp reads the 32 tensor-memory lanes of its quarter
    const int row = q * 32 + lane;
    wait_before(p);  // the row scales may be the preceding kernel's
    if constexpr (GATHER)
      gather<KIND>(p, tiles, full_bar(0), empty_bar(0), abort_flag, warp - 2, lane, m0, n0, kb0, n_kb);
    if (warp < 6 && mbar_wait_warp(done_bar, 0, abort_flag, WAIT_LIMIT_NS)) {
      tc_fence_after();
      // every MMA has read its operands: the ring's shared memory takes the accumulator
#pragma unroll 1
      for (int ch = 0; ch < 4; ch++) {
        uint32_t r[32];
        tmem_ld_32x32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(ch * 32), r);
        tmem_ld_wait();
        if (m0 + row < p.M) {
          const uint32_t dst = tiles + (uint32_t)(row * S_PITCH + ch * 32) * 4u;
#pragma unroll
          for (int j = 0; j < 8; j++)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + j * 16), "r"(r[4 * j]),
                         "r"(r[4 * j + 1]), "r"(r[4 * j + 2]), "r"(r[4 * j + 3])
                         : "memory");
        }
        __syncwarp();  // lanes of rows past M meet the others before the next load
      }
      tc_fence_before();
    } else if (warp < 6 && lane == 0) {
      report_timeout(p.status, abort_flag, 63);
    }
  }
  // warps 0 and 1 read what the preceding kernel wrote in the epilogue, too
  if (warp < 2) wait_before(p);
  if (S > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (S == 1)
    cluster_epilogue<KIND, O, ACT, THREADS, 1, 128, S_PITCH, 1>(p, tiles, rank, 0, z, m0, n0);
  else if (S == 2)
    cluster_epilogue<KIND, O, ACT, THREADS, 2, 128, S_PITCH, 1>(p, tiles, rank, 0, z, m0, n0);
  else if (S == 4)
    cluster_epilogue<KIND, O, ACT, THREADS, 4, 128, S_PITCH, 1>(p, tiles, rank, 0, z, m0, n0);
  else if (S == 8)
    cluster_epilogue<KIND, O, ACT, THREADS, 8, 128, S_PITCH, 1>(p, tiles, rank, 0, z, m0, n0);
  else
    cluster_epilogue<KIND, O, ACT, THREADS, 16, 128, S_PITCH, 1>(p, tiles, rank, 0, z, m0, n0);
  if (S > 1) cluster_sync_all();  // shared memory stays until every CTA of the cluster has read it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S_TMEM_COLS);
  }
  if (p.wait_last) grid_dep_wait();
}

// ------------------------------------------------------------------ pair kernel
constexpr int P_STAGES = 5;                       // six let the pairs drift apart in L2 (tc_gemm2.cu)
constexpr int P_STAGE_BYTES = 2 * A_TILE_BYTES;   // per CTA: 128 rows of A, its half (128) of B's columns
constexpr int P_EPI_WARPS = 8;                    // two for each tensor-memory lane quarter, half the columns each
constexpr int P_THREADS = 32 * (2 + P_EPI_WARPS);
constexpr int P_STAGING = 8192;                   // per epilogue warp: 32-row blocks, two of fp32 or four of bf16
constexpr int P_CTRL = P_STAGES * P_STAGE_BYTES + P_EPI_WARPS * P_STAGING;
constexpr int P_SMEM = P_CTRL + 1024 + 256;
static_assert(P_SMEM <= 232448, "exceeds the shared memory a CTA can opt in to");
constexpr int PN = 256;                           // accumulator columns of a tile
constexpr uint32_t P_TMEM_COLS = 512;             // two accumulators
constexpr int P_PITCH = PN + 4;                   // words between accumulator rows in shared memory, as S_PITCH
static_assert(BM * P_PITCH * 4 <= P_STAGES * P_STAGE_BYTES, "the accumulator takes the ring's place");

struct PairMaps {
  CUtensorMap a0, a1, b0, b1, c0, c1, c2;
};

// A warp's 32 x 32 block of one output, lane = row, `w` the row's packed values (two bf16 or one fp32 a word).
// With a map for C: whole rows go out through the copy engine, which clips at C's edges; shared memory is
// swizzled so that the 128-bit writes meet no bank twice.  Without (a pitch or base that TMA cannot take): rows leave
// one by one, lane = column.
template <class O, int AREA>
struct BlockStore {
  static constexpr int WORDS = sizeof(O) == 2 ? 16 : 32;
  static constexpr int BUFFERS = AREA / (32 * WORDS * 4);
  uint32_t area;  // this warp's staging
  int lane, buf = 0;

  __device__ __forceinline__ void put(const uint32_t (&w)[WORDS], const CUtensorMap* m, O* C, const Args& p, int row0,
                                      int col) {
    if (row0 >= p.M || col >= p.N) return;
    if (p.vec) {
      if (lane == 0) bulk_wait_read<BUFFERS - 1>();  // the store that last used this buffer has read it
      __syncwarp();
      const uint32_t at = area + (uint32_t)(buf * 32 * WORDS * 4);
#pragma unroll
      for (int j = 0; j < WORDS / 4; j++) {
        const int swizzled = sizeof(O) == 2 ? j ^ ((lane >> 1) & 3) : j ^ (lane & 7);
        const uint32_t dst = at + (uint32_t)(lane * WORDS * 4 + swizzled * 16);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[4 * j]), "r"(w[4 * j + 1]),
                     "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                     : "memory");
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(m, at, col, row0);
        bulk_commit();
      }
      buf = (buf + 1) % BUFFERS;
    } else {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < WORDS; j++)
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(area + (uint32_t)(lane * (WORDS + 1) + j) * 4u), "r"(w[j]) : "memory");
      __syncwarp();
      const int rows = min(32, p.M - row0);  // the same for all lanes: those past N go along and store nothing
      const bool in = col + lane < p.N;
      O* out = C + (int64_t)row0 * p.N + col + lane;
#pragma unroll 8
      for (int r = 0; r < rows; r++, out += p.N) {
        const uint32_t v = lds(area + (uint32_t)(r * (WORDS + 1) * 4 + lane * (int)sizeof(O)));
        if (!in) continue;
        if constexpr (sizeof(O) == 2)
          *reinterpret_cast<uint16_t*>(out) = (uint16_t)v;
        else
          *reinterpret_cast<uint32_t*>(out) = v;
      }
    }
    __syncwarp();  // before the warp's next load of tensor memory
  }

  static __device__ __forceinline__ uint32_t lds(uint32_t a) {  // ordered by the barriers around the block
    uint32_t v;
    if constexpr (sizeof(O) == 2)
      asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(a));
    else
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
  }
};
template <class O, int W>
__device__ __forceinline__ void pack(const float (&v)[32], uint32_t (&w)[W]) {
  if constexpr (sizeof(O) == 2) {
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; j++) w[j] = __float_as_uint(v[j]);
  }
}

// What a warp's BLOCKS blocks of 32 columns need besides the sums: a lane holds one column's scales of each block (and
// its bias), and each reaches every row of the block by a shuffle.  Loaded before the accumulator is waited for.
template <int KIND, int BLOCKS>
struct Scales {
  using T = Traits<KIND>;
  float first[T::I8 ? BLOCKS : 1], second[T::I8 ? BLOCKS : 1];

  __device__ __forceinline__ void load(const Args& p, int col, int lane) {
    if constexpr (T::I8) {
      const float* other = T::TWO ? p.col_scale1 : p.bias;
#pragma unroll
      for (int b = 0; b < BLOCKS; b++) {
        const int c = col + b * 32 + lane;
        first[b] = c < p.N ? __ldg(p.col_scale + c) : 0.f;
        second[b] = other && c < p.N ? __ldg(other + c) : 0.f;
      }
    }
  }
};

// 32 columns of one accumulator row: sums x, of the up projection y, with the scales k0 and k1 of Scales, to output
// values v; gated products leave their pre-activations in g and u.
template <int KIND, int ACT>
__device__ __forceinline__ void finish32(const uint32_t (&x)[32], const uint32_t (&y)[32], float rs, float k0, float k1,
                                         float (&v)[32], float (&g)[32], float (&u)[32]) {
  using T = Traits<KIND>;
  if constexpr (T::TWO) {
    if constexpr (T::I8) {
#pragma unroll
      for (int j = 0; j < 32; j++) {
        g[j] = scaled((int32_t)x[j], rs, __shfl_sync(0xffffffffu, k0, j));
        u[j] = scaled((int32_t)y[j], rs, __shfl_sync(0xffffffffu, k1, j));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; j++) {
        g[j] = __uint_as_float(x[j]);
        u[j] = __uint_as_float(y[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = gate<ACT>(g[j]) * u[j];
  } else if constexpr (T::I8) {
#pragma unroll
    for (int j = 0; j < 32; j++)
      v[j] = scaled((int32_t)x[j], rs, __shfl_sync(0xffffffffu, k0, j)) + __shfl_sync(0xffffffffu, k1, j);
  } else {
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = __uint_as_float(x[j]);
  }
}

// SPLIT: one tile for each cluster of two pairs; otherwise persistent over the tiles, in groups of group_rows.
template <int KIND, class O, int ACT, bool SPLIT>
__global__ void __launch_bounds__(P_THREADS, 1)
pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ Args p, int group_rows) {
  using T = Traits<KIND>;
  constexpr int BK = T::BK;
  constexpr int CN = T::TWO ? 128 : 256;  // output columns of a tile
  constexpr uint32_t IDESC = T::idesc(2 * BM, PN);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const uint32_t bars = tiles + P_CTRL;
  uint8_t* ctrl = smem_raw + (bars - raw);
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (P_STAGES + s); };
  auto tfull_bar = [&](int b) { return bars + 8u * (2 * P_STAGES + b); };
  auto tempty_bar = [&](int b) { return bars + 8u * (2 * P_STAGES + 2 + b); };
  const uint32_t slot_addr = bars + 8u * (2 * P_STAGES + 4);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl + 8 * (2 * P_STAGES + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 8 * (2 * P_STAGES + 4) + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cluster_rank = cluster_ctarank(), rank = cluster_rank & 1u;  // even: owns full[] and tempty[], issues
  const uint32_t even = cluster_rank & ~1u;
  const int split = SPLIT ? (int)(cluster_rank >> 1) : 0;
  constexpr int splits = SPLIT ? 2 : 1;
  const int pair = (int)blockIdx.x / (2 * splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < P_STAGES; s++) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 2 * P_EPI_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 2 && lane == 0) {
    prefetch_tensormap(&maps.a0);
    prefetch_tensormap(T::TWO && rank ? &maps.b1 : &maps.b0);
    prefetch_tensormap(&maps.c0);
  }
  if (warp == 1) {
    tmem_alloc2(smem_u32(const_cast<uint32_t*>(tmem_slot)), P_TMEM_COLS);
    tmem_relinquish2();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_before(p);

  const int per_z = p.tiles_m * p.tiles_n;
  const int num_tiles = per_z * (KIND == WGRAD ? 2 : 1);
  const int num_pairs = SPLIT ? num_tiles : (int)gridDim.x >> 1;  // (SPLIT: one tile for each)
  const int total = p.nkb * p.segments;
  const int kb0 = SPLIT && split ? total / 2 : 0, kb1 = SPLIT && split == 0 ? total / 2 : total;
  auto tile_coord = [&](int t, int& z, int& tm, int& tn) {
    z = t / per_z;
    t -= z * per_z;
    const int per_group = group_rows * p.tiles_n, group = t / per_group, first = group * group_rows;
    const int rows = min(group_rows, p.tiles_m - first), in_group = t - group * per_group;
    tm = first + in_group % rows;
    tn = in_group / rows;
  };
  auto give_up = [&](int where) {
    report_timeout(p.status, abort_flag, where);
    st_cluster_u32(mapa(slot_addr + 4, cluster_rank ^ 1u), 1u);  // take the partner down too
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += num_pairs) {
        int z, tm, tn;
        tile_coord(t, z, tm, tn);
        const int m0 = tm * 2 * BM + (int)rank * BM;
        const int n0 = tn * CN + (T::TWO ? 0 : (int)rank * 128);
        for (int kb = kb0; kb < kb1; kb++) {
          if (!mbar_wait_relaxed(empty_bar(stage), phase ^ 1u, abort_flag, WAIT_LIMIT_NS, 50)) {
            give_up(71);
            ok = false;
            break;
          }
          const uint32_t bar0 = mapa(full_bar(stage), even);
          const uint32_t a_dst = tiles + stage * P_STAGE_BYTES, b_dst = a_dst + A_TILE_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * P_STAGE_BYTES);
          const bool second = kb >= p.nkb;
          const int k0 = (second ? kb - p.nkb : kb) * BK;
          const CUtensorMap* ma = second || (KIND == WGRAD && z) ? &maps.a1 : &maps.a0;
          if (T::A_MN) {
            for (int c = 0; c < 2; c++) tma_load_2d_pair(a_dst + c * (A_TILE_BYTES / 2), ma, bar0, m0 + 64 * c, k0);
          } else {
            tma_load_2d_pair(a_dst, ma, bar0, k0, m0);
          }
          if (T::TWO) {
            tma_load_2d_pair(b_dst, rank ? &maps.b1 : &maps.b0, bar0, k0, n0);
          } else if (T::B_MN) {
            const CUtensorMap* mb = second ? &maps.b1 : &maps.b0;
            for (int c = 0; c < 2; c++) tma_load_2d_pair(b_dst + c * (A_TILE_BYTES / 2), mb, bar0, n0 + 64 * c, k0);
          } else {
            tma_load_2d_pair(b_dst, &maps.b0, bar0, k0, n0);
          }
          if (++stage == P_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok || *abort_flag) {  // error path: copies in flight land before the CTA leaves
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += num_pairs) {
        if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u, abort_flag, WAIT_LIMIT_NS)) {
          give_up(72);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * PN);
        for (int kb = kb0; kb < kb1; kb++) {
          if (!mbar_wait(full_bar(stage), phase, abort_flag, WAIT_LIMIT_NS)) {
            give_up(73);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = tiles + stage * P_STAGE_BYTES, b0 = a0 + A_TILE_BYTES;
          const uint64_t da = T::A_MN ? smem_desc_mn_sw128(a0, BK) : smem_desc_k_sw128(a0);
          const uint64_t db = T::B_MN ? smem_desc_mn_sw128(b0, BK) : smem_desc_k_sw128(b0);
#pragma unroll
          for (int ks = 0; ks < KSTEPS; ks++)
            tc_mma_pair<T::MMA>(d, da + ks * T::step(T::A_MN), db + ks * T::step(T::B_MN), IDESC, kb != kb0 || ks != 0);
          tc_commit_pair_at(empty_bar(stage), even);
          if (++stage == P_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit_pair_at(tfull_bar(acc), even);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    __syncwarp();
  } else if (SPLIT) {
    const int q = warp & 3, part = (warp - 2) >> 2;
    const int row = q * 32 + lane;
    if (mbar_wait_warp(tfull_bar(0), 0, abort_flag, WAIT_LIMIT_NS)) {
      tc_fence_after();
      // every MMA of this pair has read its operands: the ring takes the accumulator, for the other pairs to read
#pragma unroll 1
      for (int ch = 0; ch < 4; ch++) {
        uint32_t r[32];
        const int c = part * 128 + ch * 32;
        tmem_ld_32x32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
        tmem_ld_wait();
        const uint32_t dst = tiles + (uint32_t)(row * P_PITCH + c) * 4u;
#pragma unroll
        for (int j = 0; j < 8; j++)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + j * 16), "r"(r[4 * j]), "r"(r[4 * j + 1]),
                       "r"(r[4 * j + 2]), "r"(r[4 * j + 3])
                       : "memory");
      }
    } else if (lane == 0) {
      give_up(75);
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    BlockStore<O, P_STAGING> store{tiles + P_STAGES * P_STAGE_BYTES + (uint32_t)(warp - 2) * P_STAGING, lane};
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = pair; t < num_tiles; t += num_pairs) {
      int z, tm, tn;
      tile_coord(t, z, tm, tn);
      const int row0 = tm * 2 * BM + (int)rank * BM + q * 32, row = row0 + lane;
      const int c0 = tn * CN + part * (CN / 2);
      float rs = 0.f;
      if constexpr (T::I8)
        if (row < p.M) rs = p.row_scale[row];
      Scales<KIND, CN / 64> scales;
      scales.load(p, c0, lane);
      if (!mbar_wait_warp(tfull_bar(acc), acc_phase, abort_flag, WAIT_LIMIT_NS)) {
        if (lane == 0) give_up(74);
        break;
      }
      tc_fence_after();
      const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * PN + part * (CN / 2));
#pragma unroll
      for (int ch = 0; ch < CN / 64; ch++) {
        const int col = c0 + ch * 32;
        uint32_t x[32], y[32], w[BlockStore<O, P_STAGING>::WORDS];
        float v[32], g[32], u[32];
        tmem_ld_32x32(from + (uint32_t)(ch * 32), x);
        if constexpr (T::TWO) tmem_ld_32x32(from + (uint32_t)(128 + ch * 32), y);
        tmem_ld_wait();
        finish32<KIND, ACT>(x, y, rs, scales.first[T::I8 ? ch : 0], scales.second[T::I8 ? ch : 0], v, g, u);
        if (KIND == GATED && p.c1) {
          pack<O>(g, w);
          store.put(w, &maps.c1, static_cast<O*>(p.c1), p, row0, col);
          pack<O>(u, w);
          store.put(w, &maps.c2, static_cast<O*>(p.c2), p, row0, col);
        }
        pack<O>(v, w);
        if (KIND == WGRAD && z)
          store.put(w, &maps.c1, static_cast<O*>(p.c1), p, row0, col);
        else
          store.put(w, &maps.c0, static_cast<O*>(p.c0), p, row0, col);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(tempty_bar(acc), even));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (lane == 0) bulk_wait_all();  // shared memory outlives the stores that read it
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync_all();
  if constexpr (SPLIT) {
    int z, tm, tn;
    tile_coord(pair, z, tm, tn);
    const int m0 = tm * 2 * BM + (int)rank * BM;
    cluster_epilogue<KIND, O, ACT, P_THREADS, 2, PN, P_PITCH, 2>(p, tiles, split, (int)rank, z, m0, tn * CN);
    cluster_sync_all();  // shared memory stays until every CTA of the cluster has read it
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem, P_TMEM_COLS);
  }
  if (p.wait_last) grid_dep_wait();
}

// ------------------------------------------------------------------ tall kernel
// 512 x 256 tiles: a pair's two 256 x 256 halves share every B stage, 48 instead of 64 KiB into shared memory for the
// same products, which is what L2 and a long run under the power cap pay for (as in tc_gemm2.cu).  The two accumulators
// fill tensor memory, so nothing is left for the next tile: its upper half starts as soon as the upper accumulator has
// been read, up to three k-blocks ahead of the lower, and the epilogue reads both, as packed outputs, before it stores
// either.  Products with one weight and bf16 outputs; the gated kinds' epilogue takes too long between two tiles
// (8192 x 8192 x 4096 with kept pre-activations 900 us here, 900 on the pair kernel; int8 4096 rows 228 and 216).
constexpr int H_STAGES = 4;
constexpr int H_STAGE_BYTES = 3 * A_TILE_BYTES;  // per CTA: 2 x 128 rows of A, its half of B's columns
constexpr int H_STAGING = 4096;                  // per epilogue warp: two 32-row blocks of bf16
constexpr int H_CTRL = H_STAGES * H_STAGE_BYTES + P_EPI_WARPS * H_STAGING;
constexpr int H_SMEM = H_CTRL + 1024 + 256;
static_assert(H_SMEM <= 232448, "exceeds the shared memory a CTA can opt in to");

template <int KIND>
__global__ void __launch_bounds__(P_THREADS, 1)
tall_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ Args p, int group_rows) {
  using T = Traits<KIND>;
  using O = __nv_bfloat16;
  constexpr int BK = T::BK;
  static_assert(!T::TWO, "one weight");
  constexpr int CN = PN;
  constexpr uint32_t IDESC = T::idesc(2 * BM, PN);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const uint32_t bars = tiles + H_CTRL;
  uint8_t* ctrl = smem_raw + (bars - raw);
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (H_STAGES + s); };
  auto tfull_bar = [&](int b) { return bars + 8u * (2 * H_STAGES + b); };
  auto tempty_bar = [&](int b) { return bars + 8u * (2 * H_STAGES + 2 + b); };
  const uint32_t slot_addr = bars + 8u * (2 * H_STAGES + 4);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctrl + 8 * (2 * H_STAGES + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 8 * (2 * H_STAGES + 4) + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < H_STAGES; s++) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 2 * P_EPI_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 2 && lane == 0) {
    prefetch_tensormap(&maps.a0);
    prefetch_tensormap(&maps.b0);
    prefetch_tensormap(&maps.c0);
  }
  if (warp == 1) {
    tmem_alloc2(smem_u32(const_cast<uint32_t*>(tmem_slot)), P_TMEM_COLS);
    tmem_relinquish2();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_before(p);

  const int per_z = p.tiles_m * p.tiles_n;
  const int num_tiles = per_z * (KIND == WGRAD ? 2 : 1);
  const int total = p.nkb * p.segments;
  // This pair's items: whole tiles pair, pair + num_pairs, ... of the full rounds, then one of the rest; a rest that
  // leaves half of the pairs idle goes as half tiles (mode 1 / 2: upper / lower half alone), one a pair.
  const int full_rounds = num_tiles / num_pairs, rest = num_tiles - full_rounds * num_pairs;
  int last_tile = -1, last_mode = 0;
  if (2 * rest <= num_pairs) {
    if (pair < 2 * rest) last_tile = full_rounds * num_pairs + (pair >> 1), last_mode = 1 + (pair & 1);
  } else if (pair < rest) {
    last_tile = full_rounds * num_pairs + pair;
  }
  const int items = full_rounds + (last_tile >= 0 ? 1 : 0);
  auto item = [&](int i, int& mode, int& z, int& tm, int& tn) {
    const bool last = i == full_rounds;
    int t = last ? last_tile : pair + i * num_pairs;
    mode = last ? last_mode : 0;
    z = t / per_z;
    t -= z * per_z;
    const int per_group = group_rows * p.tiles_n, group = t / per_group, first = group * group_rows;
    const int rows = min(group_rows, p.tiles_m - first), in_group = t - group * per_group;
    tm = first + in_group % rows;
    tn = in_group / rows;
  };
  auto give_up = [&](int where) {
    report_timeout(p.status, abort_flag, where);
    st_cluster_u32(mapa(slot_addr + 4, rank ^ 1u), 1u);
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < items && ok; i++) {
        int mode, z, tm, tn;
        item(i, mode, z, tm, tn);
        const int m0 = tm * 4 * BM + (int)rank * BM + (mode == 2 ? 2 * BM : 0);  // the lower half: + 2 BM
        const int n0 = tn * CN + (int)rank * 128;
        const int halves = mode ? 1 : 2;
        for (int kb = 0; kb < total; kb++) {
          if (!mbar_wait_relaxed(empty_bar(stage), phase ^ 1u, abort_flag, WAIT_LIMIT_NS, 50)) {
            give_up(81);
            ok = false;
            break;
          }
          const uint32_t bar0 = mapa(full_bar(stage), 0);
          const uint32_t dst = tiles + stage * H_STAGE_BYTES, b_dst = dst + 2 * A_TILE_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * (halves + 1) * A_TILE_BYTES);
          const bool second = kb >= p.nkb;
          const int k0 = (second ? kb - p.nkb : kb) * BK;
          const CUtensorMap* ma = second || (KIND == WGRAD && z) ? &maps.a1 : &maps.a0;
          for (int h = 0; h < halves; h++) {
            const uint32_t a_dst = dst + h * A_TILE_BYTES;
            const int m = m0 + h * 2 * BM;
            if (T::A_MN) {
              for (int c = 0; c < 2; c++) tma_load_2d_pair(a_dst + c * (A_TILE_BYTES / 2), ma, bar0, m + 64 * c, k0);
            } else {
              tma_load_2d_pair(a_dst, ma, bar0, k0, m);
            }
          }
          if (T::B_MN) {
            const CUtensorMap* mb = second ? &maps.b1 : &maps.b0;
            for (int c = 0; c < 2; c++) tma_load_2d_pair(b_dst + c * (A_TILE_BYTES / 2), mb, bar0, n0 + 64 * c, k0);
          } else {
            tma_load_2d_pair(b_dst, &maps.b0, bar0, k0, n0);
          }
          if (++stage == H_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok || *abort_flag) {  // error path: copies in flight land before the CTA leaves
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // Two cursors into the ring: the upper half runs a k-block or more ahead of the lower, which frees the stages.
      int hi_stage = 0, lo_stage = 0;
      uint32_t hi_phase = 0, acc_phase = 0;
      bool ok = true;
      auto issue = [&](int stage, int half, bool first) {
        const uint32_t a0 = tiles + stage * H_STAGE_BYTES + half * A_TILE_BYTES;
        const uint32_t b0 = tiles + stage * H_STAGE_BYTES + 2 * A_TILE_BYTES;
        const uint64_t da = T::A_MN ? smem_desc_mn_sw128(a0, BK) : smem_desc_k_sw128(a0);
        const uint64_t db = T::B_MN ? smem_desc_mn_sw128(b0, BK) : smem_desc_k_sw128(b0);
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ks++)
          tc_mma_pair<T::MMA>(tmem + (uint32_t)(half * PN), da + ks * T::step(T::A_MN), db + ks * T::step(T::B_MN), IDESC,
                              !(first && ks == 0));
      };
      auto upper = [&](int kb) -> bool {
        if (!mbar_wait(full_bar(hi_stage), hi_phase, abort_flag, WAIT_LIMIT_NS)) {
          give_up(82);
          return false;
        }
        tc_fence_after();
        issue(hi_stage, 0, kb == 0);
        if (++hi_stage == H_STAGES) {
          hi_stage = 0;
          hi_phase ^= 1u;
        }
        return true;
      };
      for (int i = 0; i < items && ok; i++) {
        int mode, z, tm, tn;
        item(i, mode, z, tm, tn);
        if (!mbar_wait(tempty_bar(0), acc_phase ^ 1u, abort_flag, WAIT_LIMIT_NS)) {
          give_up(83);
          break;
        }
        tc_fence_after();
        if (mode) {  // always this pair's last item: one accumulator, stages freed at once
          for (int kb = 0; kb < total && ok; kb++) {
            const int stage = hi_stage;
            ok = upper(kb);
            if (ok) tc_commit_pair(empty_bar(stage));
          }
          if (ok) tc_commit_pair(tfull_bar(0));
          break;
        }
        int hi = 0;  // k-blocks that the upper half has had
        while (ok && hi < total && hi < H_STAGES - 1 && (hi < 1 || !mbar_try_wait(tempty_bar(1), acc_phase ^ 1u))) {
          ok = upper(hi++);
          if (ok && hi == total) tc_commit_pair(tfull_bar(0));
        }
        if (!ok) break;
        if (!mbar_wait(tempty_bar(1), acc_phase ^ 1u, abort_flag, WAIT_LIMIT_NS)) {
          give_up(84);
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < total; kb++) {
          if (hi < total && hi - kb <= 1) {
            if (!upper(hi++)) {
              ok = false;
              break;
            }
            if (hi == total) tc_commit_pair(tfull_bar(0));
          }
          issue(lo_stage, 1, kb == 0);  // its stage was waited for when the upper half used it
          tc_commit_pair(empty_bar(lo_stage));
          if (++lo_stage == H_STAGES) lo_stage = 0;
        }
        if (!ok) break;
        tc_commit_pair(tfull_bar(1));
        acc_phase ^= 1u;
      }
    }
    __syncwarp();
  } else {
    constexpr int BLOCKS = CN / 64;                    // 32-column blocks of this warp in a half: its half of the columns
    const int q = warp & 3, part = (warp - 2) >> 2;
    BlockStore<O, H_STAGING> store{tiles + H_STAGES * H_STAGE_BYTES + (uint32_t)(warp - 2) * H_STAGING, lane};
    uint32_t acc_phase = 0;
    // an accumulator's share of this warp as packed outputs; the accumulator goes back to the MMA thread
    auto take = [&](int half, int row, int c0, uint32_t (&w)[BLOCKS][16]) -> bool {
      float rs = 0.f;
      if constexpr (T::I8)
        if (row < p.M) rs = p.row_scale[row];
      Scales<KIND, BLOCKS> scales;
      scales.load(p, c0, lane);
      if (!mbar_wait_warp(tfull_bar(half), acc_phase, abort_flag, WAIT_LIMIT_NS)) {
        if (lane == 0) give_up(85);
        return false;
      }
      tc_fence_after();
      const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * PN + part * (CN / 2));
#pragma unroll
      for (int b = 0; b < BLOCKS; b++) {
        uint32_t x[32];
        float v[32];
        tmem_ld_32x32(from + (uint32_t)(b * 32), x);
        tmem_ld_wait();
        finish32<KIND, 0>(x, x, rs, scales.first[T::I8 ? b : 0], scales.second[T::I8 ? b : 0], v, v, v);
        pack<O>(v, w[b]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(tempty_bar(half), 0));
      return true;
    };
    auto put = [&](const uint32_t (&w)[BLOCKS][16], int z, int row0, int c0) {
      const bool second = KIND == WGRAD && z;
#pragma unroll
      for (int b = 0; b < BLOCKS; b++)
        store.put(w[b], second ? &maps.c1 : &maps.c0, static_cast<O*>(second ? p.c1 : p.c0), p, row0, c0 + b * 32);
    };
    for (int i = 0; i < items; i++) {
      int mode, z, tm, tn;
      item(i, mode, z, tm, tn);
      const int c0 = tn * CN + part * (CN / 2);
      const int upper0 = tm * 4 * BM + (int)rank * BM + q * 32 + (mode == 2 ? 2 * BM : 0), lower0 = upper0 + 2 * BM;
      uint32_t upper[BLOCKS][16], lower[BLOCKS][16];
      if (!take(0, upper0 + lane, c0, upper)) break;
      if (mode) {
        put(upper, z, upper0, c0);
        break;
      }
      if (!take(1, lower0 + lane, c0, lower)) break;
      put(upper, z, upper0, c0);
      put(lower, z, lower0, c0);
      acc_phase ^= 1u;
    }
    if (lane == 0) bulk_wait_all();  // shared memory outlives the stores that read it
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem, P_TMEM_COLS);
  }
  if (p.wait_last) grid_dep_wait();
}

// ------------------------------------------------------------------ operand copies with a pitch that TMA takes
// TMA reads rows whose pitch and base are multiples of 16 bytes.  Other operands are multiplied from copies with the
// pitch rounded up; each thread assembles 16 bytes from the two aligned vectors around them (bytes behind the row's end
// are whatever lies there; the tensor map ends before them).
struct PadJob {
  const uint8_t* src;
  uint8_t* dst;
  int64_t rows, src_pitch, dst_pitch;
};
constexpr int kMaxPads = 5;
struct PadJobs {
  PadJob job[kMaxPads];
};

__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ PadJobs jobs) {
  const PadJob& j = jobs.job[blockIdx.y];
  const int64_t per_row = j.dst_pitch / 16, n = j.rows * per_row;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    // (a 64-bit division would take longer than the copy)
    const int64_t r = n <= UINT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row;
    const int64_t c = (i - r * per_row) * 16;
    const uint8_t* s = j.src + r * j.src_pitch + c;
    const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(s) & 15u);
    const uint4* v = reinterpret_cast<const uint4*>(s - shift);
    const uint4 lo = __ldg(v);
    // the second only where it holds a byte of the row
    const uint4 hi = j.src_pitch - c > 16 - (int)shift ? __ldg(v + 1) : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(j.dst + r * j.dst_pitch + c) = join16(lo, hi, shift);
  }
}

// Memory of one call, ordered on its stream: freed behind the call's kernels, and inside a graph when the call is
// captured, so that neither other streams nor other graphs ever see it.
class StreamMemory {
 public:
  StreamMemory(exo_b200_Context* ctx) : ctx_(ctx) {}
  ~StreamMemory() {
    if (p_) cudaFreeAsync(p_, ctx_->stream);
  }
  StreamMemory(const StreamMemory&) = delete;
  StreamMemory& operator=(const StreamMemory&) = delete;
  cudaError_t get(size_t bytes) {
    if (!ctx_->pool) {
      cudaMemPoolProps props = {};
      props.allocType = cudaMemAllocationTypePinned;
      props.location.type = cudaMemLocationTypeDevice;
      props.location.id = ctx_->device;
      cudaError_t e = cudaMemPoolCreate(&ctx_->pool, &props);
      if (e != cudaSuccess) {
        ctx_->pool = nullptr;
        return e;
      }
      // Freed blocks stay for the next call, until exo_b200_context_trim: going back at every synchronisation they would
      // be mapped anew in the call after it (64 x 16384 x 4095 gated, 268 MB of copies: 155 us, 2 to 4 ms when mapped).
      uint64_t keep = UINT64_MAX;
      cudaMemPoolSetAttribute(ctx_->pool, cudaMemPoolAttrReleaseThreshold, &keep);
    }
    cudaError_t e = cudaMallocFromPoolAsync(&p_, bytes, ctx_->pool, ctx_->stream);
    if (e != cudaSuccess) p_ = nullptr;
    return e;
  }
  uint8_t* data() const { return static_cast<uint8_t*>(p_); }

 private:
  exo_b200_Context* ctx_;
  void* p_ = nullptr;
};

// One operand: rows of `width` elements.
struct Matrix {
  const void* base;
  int64_t rows, width, pitch;  // pitch in bytes
};

// Copies the operands that TMA cannot read; `copied` says whether any was.
cudaError_t make_readable(exo_b200_Context* ctx, StreamMemory& memory, int elem, Matrix* const* ops, int n,
                          bool* copied) {
  PadJobs jobs;
  int count = 0;
  size_t bytes = 0;
  int64_t most = 0;
  int which[kMaxPads];
  for (int i = 0; i < n; i++) {
    Matrix& m = *ops[i];
    if (m.pitch % 16 == 0 && aligned16(m.base)) continue;
    const int64_t pitch = (m.width * elem + 15) / 16 * 16;
    jobs.job[count] = PadJob{static_cast<const uint8_t*>(m.base), nullptr, m.rows, m.width * elem, pitch};
    which[count++] = i;
    bytes += (size_t)(m.rows * pitch);
    most = std::max(most, m.rows * pitch / 16);
  }
  *copied = count > 0;
  if (!count) return cudaSuccess;
  cudaError_t e = memory.get(bytes);
  if (e != cudaSuccess) return e;
  uint8_t* at = memory.data();
  for (int c = 0; c < count; c++) {
    jobs.job[c].dst = at;
    ops[which[c]]->base = at;
    ops[which[c]]->pitch = jobs.job[c].dst_pitch;
    at += jobs.job[c].rows * jobs.job[c].dst_pitch;
  }
  const unsigned grid = (unsigned)std::min<int64_t>((most + 255) / 256, (int64_t)ctx->sm_count * 16);
  pad_rows_kernel<<<dim3(grid, (unsigned)count), 256, 0, ctx->stream>>>(jobs);
  return cudaGetLastError();
}

bool map_of(CUtensorMap* m, const Matrix& x, int elem, int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)x.width, (cuuint64_t)x.rows};
  cuuint64_t strides[1] = {(cuuint64_t)x.pitch};
  cuuint32_t box[2] = {(cuuint32_t)(ROW_BYTES / elem), (cuuint32_t)box_rows};
  return encode_tiled_map(m, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x.base,
                          dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

#define EXOB200_CLUSTER16_ONCE(kernel, device)                                                                        \
  do {                                                                                                                \
    static std::atomic<uint64_t> done_{0};                                                                            \
    const uint64_t bit_ = 1ull << ((device) & 63);                                                                    \
    if (!(done_.load(std::memory_order_acquire) & bit_)) {                                                            \
      cudaError_t e_ = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);               \
      if (e_ != cudaSuccess) return e_;                                                                               \
      done_.fetch_or(bit_, std::memory_order_release);                                                                \
    }                                                                                                                 \
  } while (0)

// How many clusters of 2, 4, 8 and 16 CTAs of the split kernel the GPU holds at once with an SM for each CTA: fewer than
// its SMs would make, since a cluster stays within one group of them.  Asked once per context, of one instance.
cudaError_t ask_clusters(exo_b200_Context* ctx) {
  auto* kernel = split_kernel<DGRAD, __nv_bfloat16, 0, false>;
  EXOB200_SMEM_ATTR_ONCE(kernel, S_SMEM_ALONE, ctx->device);
  EXOB200_CLUSTER16_ONCE(kernel, ctx->device);
  for (int i = 0; i < 4; i++) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2u << i;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(2u << i);
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.dynamicSmemBytes = S_SMEM_ALONE;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&ctx->ffn_clusters[i], kernel, &cfg);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
// Whether `tiles` clusters of 2^(i + 1) CTAs run at once.
bool clusters_fit(exo_b200_Context* ctx, int64_t tiles, int i) {
  if (ctx->ffn_clusters[0] == 0 && ask_clusters(ctx) != cudaSuccess) {
    cudaGetLastError();
    for (int k = 0; k < 3; k++) ctx->ffn_clusters[k] = ctx->sm_count / (4 << k);
    ctx->ffn_clusters[3] = 0;
  }
  return tiles <= ctx->ffn_clusters[i];
}

// How many CTAs of the split kernel share a tile's reduction: as long as every CTA has an SM to itself, at once, and two
// k-blocks.  Past one CTA for each SM, and mostly past four of them on one tile, adding up costs more than the shorter
// loops save: 256 x 2048 x 4096 int8 (32 tiles) 14.3, 10.5, 9.5 and 14.8 us with 1, 2, 4 and 8 CTAs a tile;
// 512 x 2048 x 4096 (64 tiles) 14.7, 11.0, 13.0 and 26.7; 16 x 4480 x 4096 (35 tiles, whose clusters of four do not run
// at once) 9.2 with two, 13.0 with four.  A handful of tiles with a long reduction splits further (the gradient of 3 x 177
// inputs over 2 x 14054 units, two tiles: 33 us of a 60 us backward pass with four, 12.8 with sixteen).
int split_of(exo_b200_Context* ctx, int64_t tiles, int k_blocks) {
  int S = 1, i = 0;
  for (; S < 4 && clusters_fit(ctx, tiles, i) && k_blocks / (2 * S) >= 2; i++) S *= 2;
  for (; S >= 4 && S < MAX_SPLIT && tiles * S * 4 <= ctx->sm_count && clusters_fit(ctx, tiles, i) &&
         k_blocks / (2 * S) >= 8; i++)
    S *= 2;
  return S;
}

// Which kernel: 0 the split kernel, 1 the persistent pair kernel, 2 the pair kernel with its reduction split over two
// pairs.  EXOB200_FFN_PAIR=0 / 1 / 2 forces it.
// Up to 128 rows the weights' bytes are what counts, and the split kernel's CTAs share them out more evenly
// (1 x 16384 x 4096 gated: 47 against 73 us).  Above, a pair's 256 x 256 tile moves half the operand bytes of four
// 128 x 128 tiles, which come no faster than 14 TB/s out of L2 (8192^3 int8: 345 against 526 us).  Below a full round
// of tiles the time is a fixed part and so much for each k-block that one CTA goes through: fitted, in us, on products
// and gated products of 160 to 2048 rows, 512 to 8192 columns and 2 to 64 k-blocks (split / pair / two pairs measured:
// 1024 x 1024 x 1024 int8 7.6 / 9.5 / 9.3, 1024 x 4096 x 4096 19.9 / 19.1 / 28, 512 x 4096 x 4096 15.9 / 17.0 / 14.0).
int pair_splits(exo_b200_Context* ctx, int64_t rows, int64_t pair_tiles, int64_t split_tiles, int k_blocks) {
  static const int mode = [] {
    const char* e = getenv("EXOB200_FFN_PAIR");
    return e ? atoi(e) : -1;
  }();
  if (mode >= 0) return std::min(std::min(mode, 2), k_blocks);
  if (rows <= 128) return 0;
  const int S = split_of(ctx, split_tiles, k_blocks), sms = ctx->sm_count, pairs = sms / 2;
  auto rounds = [](int64_t work, int64_t slots) { return (double)((work + slots - 1) / slots); };
  const bool alone = split_tiles * S <= sms;
  const double loop = rounds(k_blocks, S);
  const double turns = rounds(split_tiles, 2 * sms);  // of CTAs that share SMs; each ends in an epilogue of its own
  const double split = 5.2 + (alone ? 0.30 * loop + (S > 1 ? 0.5 : 0.0) : 0.46 * loop * turns + 5.0 * (turns - 1.0));
  const double pair = 6.0 + 0.31 * k_blocks * rounds(pair_tiles, pairs);
  const double two = clusters_fit(ctx, pair_tiles, 1) && k_blocks >= 2 ? 8.0 + 0.34 * rounds(k_blocks, 2) : 1e30;
  return split <= pair && split <= two ? 0 : pair <= two ? 1 : 2;
}

// Operands that TMA cannot read: gathered as they are, or copied first.  Measured, gathered / copied: 16 x 16384 x 4095
// gated bf16 95 / 141 us, int8 51 / 72, 16 x 4099 x 4099 int8 15.1 / 15.9, small ones 1 to 2 us slower on the GPU but
// 3 us less for the host, which has neither memory to order nor a second launch; with 64 tokens 174 / 142 us.
// EXOB200_FFN_GATHER=0 switches it off.
bool gather_wanted(int64_t rows) {
  static const bool off = [] {
    const char* e = getenv("EXOB200_FFN_GATHER");
    return e && e[0] == '0';
  }();
  return !off && rows <= G_MAX_M;
}

template <int KIND, class O, int ACT, bool GATHER>
cudaError_t launch_split(exo_b200_Context* ctx, const CUtensorMap (&maps)[4], const Args& a, int64_t tiles,
                         bool after_own_kernel) {
  auto* kernel = split_kernel<KIND, O, ACT, GATHER>;
  EXOB200_SMEM_ATTR_ONCE(kernel, GATHER ? G_SMEM : S_SMEM_ALONE, ctx->device);
  const int total = a.nkb * a.segments;
  const int S = split_of(ctx, tiles, total);
  if (tiles * S > INT32_MAX) return cudaErrorInvalidValue;
  if (S > 8) EXOB200_CLUSTER16_ONCE(kernel, ctx->device);
  const int stage_bytes = (Traits<KIND>::A_MN ? A_TILE_BYTES : a.a_rows * ROW_BYTES) + A_TILE_BYTES;
  const int room = (tiles * S <= ctx->sm_count ? S_SMEM_ALONE : S_SMEM_SHARED) - S_CTRL;
  const int stages = std::min(S_MAX_STAGES, room / stage_bytes);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * S));
  cfg.blockDim = dim3(GATHER ? G_THREADS : NUM_THREADS);
  cfg.dynamicSmemBytes = GATHER ? G_SMEM : stages * stage_bytes + S_CTRL;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (S > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)S;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    n++;
  }
  if (after_own_kernel && dependent_launches()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], maps[3], a, S, stages);
}

// A kernel of CTA pairs, `splits` pairs to a cluster; persistent ones on as many pairs as fit the GPU.
template <class Kernel>
cudaError_t launch_pairs(exo_b200_Context* ctx, Kernel* kernel, int smem, const PairMaps& maps, const Args& a,
                         int64_t tiles, int splits, int group_rows, bool after_own_kernel) {
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(P_THREADS);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * (unsigned)splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (splits > 1) {
    cfg.gridDim = dim3(2 * (unsigned)(tiles * splits));
  } else {
    // every instance takes a whole SM, so all of them fit as many pairs; asked once per context
    int& max_pairs = ctx->max_ffn_pairs;
    if (max_pairs == 0) {
      cfg.gridDim = dim3(2 * ctx->sm_count);
      int n = 0;
      cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      if (e != cudaSuccess) return e;
      max_pairs = std::max(1, n);
    }
    cfg.gridDim = dim3(2 * (unsigned)std::min<int64_t>(tiles, max_pairs));
  }
  if (after_own_kernel && dependent_launches()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kernel, maps, a, group_rows);
}

template <int KIND, class O, int ACT, bool SPLIT>
cudaError_t launch_pair(exo_b200_Context* ctx, const PairMaps& maps, const Args& a, int64_t tiles,
                        bool after_own_kernel) {
  auto* kernel = pair_kernel<KIND, O, ACT, SPLIT>;
  EXOB200_SMEM_ATTR_ONCE(kernel, P_SMEM, ctx->device);
  return launch_pairs(ctx, kernel, P_SMEM, maps, a, tiles, SPLIT ? 2 : 1, 8, after_own_kernel);
}

template <int KIND>
cudaError_t launch_tall(exo_b200_Context* ctx, const PairMaps& maps, const Args& a, int64_t tiles,
                        bool after_own_kernel) {
  auto* kernel = tall_kernel<KIND>;
  EXOB200_SMEM_ATTR_ONCE(kernel, H_SMEM, ctx->device);
  return launch_pairs(ctx, kernel, H_SMEM, maps, a, tiles, 1, 6, after_own_kernel);
}

// The tall kernel where the pair kernel would run unsplit: with tiles for three pairs of four and a reduction that outlasts
// the change from tile to tile.  Measured over 0.15 s runs, tall / pair: gradients of 8192 x 8192 x 4096 1785 / 1935 us,
// of 4096 x 4096 x 2048 256 / 270; int8 8192^3 398 / 412, 4096^3 (32 k-blocks) 63.5 / 62.8, 4096 x 8192 x 1024 45.1 / 43.8.
// EXOB200_FFN_TALL=0 / 1 forces it off / on.
bool tall_wanted(const exo_b200_Context* ctx, int64_t tall_tiles, int k_blocks) {
  static const int mode = [] {
    const char* e = getenv("EXOB200_FFN_TALL");
    return e ? atoi(e) : -1;
  }();
  return mode >= 0 ? mode == 1 : k_blocks >= 48 && tall_tiles * 8 >= 3 * ctx->sm_count;
}

// Tensor map of a dense output for 32 x 32 blocks out of swizzled shared memory
template <class O>
bool output_map(CUtensorMap* m, void* base, int64_t rows, int64_t cols) {
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols * sizeof(O)};
  cuuint32_t box[2] = {32, 32};
  return encode_tiled_map(m, sizeof(O) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2,
                          base, dims, strides, box,
                          sizeof(O) == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

// How a product stands to the kernel before it on the stream.
enum After {
  OTHERS,  // anything: wait for it in the ordinary way
  OWN,     // a kernel of the same call, itself ordered after everything earlier: this one may be scheduled beside it and
           // waits for it before reading what it writes
  BESIDE   // a product that was launched OWN and let its successors start: this one reads nothing of it, runs beside it
           // and only ends after it
};

template <int KIND, class O, int ACT>
cudaError_t run(exo_b200_Context* ctx, const Problem& p, const Matrix& a0, const Matrix& a1, const Matrix& b0,
                const Matrix& b1, After after, bool b_copied, bool let_beside) {
  using T = Traits<KIND>;
  constexpr int E = T::ELEM;
  constexpr bool USES_A1 = KIND == WGRAD || KIND == DGRAD, USES_B1 = T::TWO || KIND == DGRAD;
  Args a{};
  a.M = (int)p.M, a.N = (int)p.N;
  a.nkb = (int)((p.K + T::BK - 1) / T::BK);
  a.segments = KIND == DGRAD ? 2 : 1;
  a.row_scale = p.row_scale, a.col_scale = p.col_scale, a.col_scale1 = p.col_scale1, a.bias = p.bias;
  a.c0 = p.c0, a.c1 = p.c1, a.c2 = p.c2;
  a.status = ctx->status_dev;
  a.b_early = after == OWN && !b_copied;
  a.wait_last = after == BESIDE;
  a.let_beside = let_beside;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.c0) | reinterpret_cast<uintptr_t>(p.c1) |
                         reinterpret_cast<uintptr_t>(p.c2);
  const int Z = KIND == WGRAD ? 2 : 1;
  auto tiles_of = [&](int64_t rows, int64_t cols) {
    a.tiles_m = (int)((p.M + rows - 1) / rows);
    a.tiles_n = (int)((p.N + cols - 1) / cols);
    return (int64_t)a.tiles_m * a.tiles_n * Z;
  };
  const bool any4 = p.N % 4 == 0 && bits % (4 * sizeof(O)) == 0;  // four columns at a time
  if constexpr (!T::B_MN) {
    auto readable = [](const Matrix& m) { return m.pitch % 16 == 0 && aligned16(m.base); };
    if (!(readable(a0) && readable(b0) && (!USES_B1 || readable(b1)))) {  // only left as they are to be gathered
      const int64_t tiles = tiles_of(BM, T::TWO ? 64 : 128);
      if (tiles > INT32_MAX) return cudaErrorInvalidValue;
      a.a_rows = (int)std::min<int64_t>(BM, (p.M + 7) / 8 * 8);
      a.vec = any4;
      a.a = static_cast<const uint8_t*>(a0.base);
      a.b = static_cast<const uint8_t*>(b0.base), a.b1 = static_cast<const uint8_t*>(b1.base);
      a.row_bytes = (int)(p.K * E);
      CUtensorMap none[4] = {};
      return launch_split<KIND, O, ACT, true>(ctx, none, a, tiles, after != OTHERS);
    }
  }
  const int64_t split_tiles = tiles_of(BM, T::TWO ? 64 : 128);
  const int64_t pair_tiles = tiles_of(2 * BM, T::TWO ? 128 : 256);
  if (split_tiles > INT32_MAX) return cudaErrorInvalidValue;
  const int splits = pair_splits(ctx, p.M, pair_tiles, split_tiles, a.nkb * a.segments);
  const int b_box = T::B_MN ? T::BK : T::TWO && !splits ? 64 : 128;
  if (splits) {
    a.vec = splits > 1 ? any4 : p.N * (int64_t)sizeof(O) % 16 == 0 && bits % 16 == 0;
    PairMaps m;
    if (!map_of(&m.a0, a0, E, T::A_MN ? T::BK : BM)) return cudaErrorUnknown;
    m.a1 = m.a0;
    if (USES_A1 && !map_of(&m.a1, a1, E, T::A_MN ? T::BK : BM)) return cudaErrorUnknown;
    if (!map_of(&m.b0, b0, E, b_box)) return cudaErrorUnknown;
    m.b1 = m.b0;
    if (USES_B1 && !map_of(&m.b1, b1, E, b_box)) return cudaErrorUnknown;
    m.c0 = m.c1 = m.c2 = m.a0;
    if (a.vec && splits == 1 &&
        !(output_map<O>(&m.c0, p.c0, p.M, p.N) && (!p.c1 || output_map<O>(&m.c1, p.c1, p.M, p.N)) &&
          (!p.c2 || output_map<O>(&m.c2, p.c2, p.M, p.N))))
      return cudaErrorUnknown;
    if constexpr (!T::TWO && sizeof(O) == 2) {
      const int64_t tall_tiles = tiles_of(4 * BM, PN);
      if (splits == 1 && tall_wanted(ctx, tall_tiles, a.nkb * a.segments))
        return launch_tall<KIND>(ctx, m, a, tall_tiles, after != OTHERS);
      tiles_of(2 * BM, PN);
    }
    return splits > 1 ? launch_pair<KIND, O, ACT, true>(ctx, m, a, pair_tiles, after != OTHERS)
                      : launch_pair<KIND, O, ACT, false>(ctx, m, a, pair_tiles, after != OTHERS);
  }
  tiles_of(BM, T::TWO ? 64 : 128);
  a.a_rows = (int)std::min<int64_t>(BM, (p.M + 7) / 8 * 8);
  a.vec = any4;
  CUtensorMap maps[4];
  if (!map_of(&maps[0], a0, E, T::A_MN ? T::BK : a.a_rows)) return cudaErrorUnknown;
  maps[1] = maps[0];
  if (USES_A1 && !map_of(&maps[1], a1, E, T::A_MN ? T::BK : a.a_rows)) return cudaErrorUnknown;
  if (!map_of(&maps[2], b0, E, b_box)) return cudaErrorUnknown;
  maps[3] = maps[2];
  if (USES_B1 && !map_of(&maps[3], b1, E, b_box)) return cudaErrorUnknown;
  return launch_split<KIND, O, ACT, false>(ctx, maps, a, split_tiles, after != OTHERS);
}

// The forward kinds: A [M,K], B [N,K].
template <int KIND, class O, int ACT>
cudaError_t launch(exo_b200_Context* ctx, const Problem& p, bool after_own_kernel) {
  using T = Traits<KIND>;
  constexpr int E = T::ELEM;
  Matrix a0{p.a0, p.M, p.K, p.K * E}, b0{p.b0, p.N, p.K, p.K * E}, b1 = b0;
  b1.base = p.b1;
  StreamMemory memory(ctx);
  bool copied = false;
  if (!(gather_wanted(p.M) && p.K * E < INT32_MAX - 1024)) {
    Matrix* ops[3] = {&a0, &b0, &b1};
    const cudaError_t e = make_readable(ctx, memory, E, ops, T::TWO ? 3 : 2, &copied);
    if (e != cudaSuccess) return e;
  }
  return run<KIND, O, ACT>(ctx, p, a0, a0, b0, b1, after_own_kernel || copied ? OWN : OTHERS, copied, false);
}

}  // namespace

cudaError_t launch_product(exo_b200_Context* ctx, Kind kind, bool out_f32, const Problem& p, bool after_own_kernel) {
  using bf16 = __nv_bfloat16;
  const bool own = after_own_kernel;
  if (rows_wanted(kind, p)) return launch_rows(ctx, kind, out_f32, p, own);
  switch (kind) {
    case SCALED:
      return out_f32 ? launch<SCALED, float, 0>(ctx, p, own) : launch<SCALED, bf16, 0>(ctx, p, own);
    case GATED:
      return p.act == 0   ? launch<GATED, bf16, 0>(ctx, p, own)
             : p.act == 1 ? launch<GATED, bf16, 1>(ctx, p, own)
                          : launch<GATED, bf16, 2>(ctx, p, own);
    case GATED_I8:
      return p.act == 0   ? launch<GATED_I8, bf16, 0>(ctx, p, own)
             : p.act == 1 ? launch<GATED_I8, bf16, 1>(ctx, p, own)
                          : launch<GATED_I8, bf16, 2>(ctx, p, own);
    default:
      return cudaErrorInvalidValue;  // the backward kinds go through launch_gradients
  }
}

cudaError_t launch_gradients(exo_b200_Context* ctx, int64_t M, int64_t F, int64_t K, const void* X, const void* Wg,
                             const void* Wu, const void* dG, const void* dU, void* dX, void* dWg, void* dWu) {
  using bf16 = __nv_bfloat16;
  Matrix dg{dG, M, F, F * 2}, du{dU, M, F, F * 2}, x{X, M, K, K * 2}, wg{Wg, F, K, K * 2}, wu{Wu, F, K, K * 2};
  // one pass of copies serves both products
  Matrix* ops[5];
  int n = 0;
  if (dX || dWg) ops[n++] = &dg, ops[n++] = &du;
  if (dX) ops[n++] = &wg, ops[n++] = &wu;
  if (dWg) ops[n++] = &x;
  StreamMemory memory(ctx);
  bool copied = false;
  cudaError_t e = make_readable(ctx, memory, 2, ops, n, &copied);
  if (e == cudaSuccess && dX) {
    Problem p{};
    p.M = M, p.N = K, p.K = F;
    p.c0 = dX;
    e = run<DGRAD, bf16, 0>(ctx, p, dg, du, wg, wu, OWN, copied, dWg != nullptr);
  }
  if (e == cudaSuccess && dWg) {
    Problem p{};
    p.M = F, p.N = K, p.K = M;
    p.c0 = dWg, p.c1 = dWu;
    e = run<WGRAD, bf16, 0>(ctx, p, dg, du, x, x, dX ? BESIDE : OWN, copied, false);
  }
  return e;
}

}  // namespace ffn
}  // namespace exob200
