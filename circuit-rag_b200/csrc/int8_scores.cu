// Products of 8-bit queries with 8-bit rows (circuit_op_int8_scores):
// out[i][j] = sq_i sr_j sum_k q_ik c_jk + bias_j, the sum exact in 32-bit integers.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "engine.h"
#include "int8.cuh"
#include "tcgen05.cuh"

namespace cb {
namespace i8 {

struct ScoresParams {
  const int8_t* q;
  const float* q_scales;
  const int8_t* codes;
  const float* scales;
  const float* bias;  // nullptr: none
  void* out;
  int64_t nq, n, q_stride, code_stride, out_stride;
  int d;
  int pairs;  // two neighbouring 16-bit results of a row of `out` may be stored as one
};

__device__ __forceinline__ float result(int acc, float sq, float sr, float bias) {
  return fmaf((float)acc * sq, sr, bias);
}

// ---------------------------------------------------------------- few bytes
// One or two queries against few rows: latency.  Eight lanes a row, each with 16
// codes a step, the queries in shared memory (zero past d, so what a row's padding
// holds does not count).
template <typename T, int NQ>
__global__ void __launch_bounds__(256) k_scores_rows(ScoresParams P) {
  griddep_wait();
  griddep_launch();
  extern __shared__ __align__(16) int8_t s_q[];
  const int chunks = (P.d + 15) >> 4;
  const int64_t q0 = (int64_t)blockIdx.y * NQ;
  for (int i = threadIdx.x; i < NQ * chunks * 16; i += blockDim.x) {
    const int q = i / (chunks * 16), c = i - q * (chunks * 16);
    s_q[i] = q0 + q < P.nq && c < P.d ? P.q[(q0 + q) * P.q_stride + c] : (int8_t)0;
  }
  __syncthreads();
  const int sub = threadIdx.x & 7;
  const int64_t groups = (int64_t)gridDim.x * (blockDim.x >> 3);
  // whole warps stay in the loop together: the shuffles need every lane
  for (int64_t row0 = (blockIdx.x * (int64_t)blockDim.x + (threadIdx.x & ~31)) >> 3; row0 < P.n; row0 += groups) {
    const int64_t row = row0 + ((threadIdx.x & 31) >> 3);
    const bool live = row < P.n;
    const int4* r = reinterpret_cast<const int4*>(P.codes + (live ? row : 0) * P.code_stride);
    int acc[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) acc[q] = 0;
    for (int c = sub; c < chunks; c += 8) {
      const int4 b = r[c];
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int4 a = reinterpret_cast<const int4*>(s_q)[q * chunks + c];
        acc[q] = __dp4a(a.x, b.x, __dp4a(a.y, b.y, __dp4a(a.z, b.z, __dp4a(a.w, b.w, acc[q]))));
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) acc[q] += __shfl_xor_sync(FULL_MASK, acc[q], o);
      if (live && sub == (q & 7) && q0 + q < P.nq)
        reinterpret_cast<T*>(P.out)[(q0 + q) * P.out_stride + row] =
            RowType<T>::put(result(acc[q], P.q_scales[q0 + q], P.scales[row], P.bias ? P.bias[row] : 0.f));
    }
  }
}

// ---------------------------------------------------------------- tensor-core products
// One persistent CTA an SM.  A unit is 128 rows (the MMA's M) against BN queries
// (its N); units are dealt round robin with the query tiles fastest, so a row
// tile comes from HBM once and its other query tiles read it from L2.  A TMA warp
// streams 128-byte K chunks of both operands through a ring of stages, one elected
// thread issues the MMAs into one of two to eight TMEM accumulators, and sixteen
// epilogue warps scale the others.  With rows as M, a lane of the accumulator is a row
// and a column a query: each warp store writes 32 consecutive results of one
// query's row of `out`, without a transposition.
constexpr int MMA_ROWS = 128;
// Epilogue warps: four cover a tile's 128 TMEM lanes and `parts` of them its columns; for
// few queries `groups` of them take turns with the tiles, since what a small tile
// costs is the way from the MMA through the accumulator to the stores (about 1,800
// clocks with one group and two accumulators), not its results.  Then a TMA and an
// MMA warp.
constexpr int EPILOGUE_WARPS = 16;
constexpr int MMA_THREADS = (EPILOGUE_WARPS + 2) * 32;
constexpr int column_parts(int BN) { return BN <= 64 ? 1 : BN / 64; }
constexpr int tile_groups(int BN) { return EPILOGUE_WARPS / 4 / column_parts(BN); }
// Accumulators of SUBS x BN columns in 512 columns of TMEM.  SUBS: 128-row tiles of a
// unit.  A unit's way through the MMA warp (two waits, two commits) takes 800 clocks
// however little it is, so with rows of one chunk two tiles go as one unit
// (4M rows of 64, 8 queries: 107 -> 74 us).
constexpr int accumulators(int BN, int SUBS = 1) { return 512 / (BN * SUBS) < 8 ? 512 / (BN * SUBS) : 8; }

// Units first, first + step, ... as (row tile, query tile), query tiles fastest,
// without a division a unit.
struct Units {
  int64_t u, step, rt, step_rt;
  int qt, step_qt, q_tiles;
  __device__ __forceinline__ Units(int64_t first, int64_t by, int tiles)
      : u(first), step(by), rt(first / tiles), step_rt(by / tiles), qt((int)(first % tiles)), step_qt((int)(by % tiles)),
        q_tiles(tiles) {}
  __device__ __forceinline__ void next() {
    u += step;
    rt += step_rt;
    qt += step_qt;
    if (qt >= q_tiles) {
      qt -= q_tiles;
      ++rt;
    }
  }
};

constexpr int RING_BYTES = 192 * 1024;
// Rows in flight: 96 KB an SM is best (2M rows of 384, one query: 3 / 4 / 5 / 6 / 8 / 12
// stages of 16 KB take 146 / 129 / 123 / 117 / 117 / 123 us; 32 queries: 184 / 163 / 158 /
// 153 / 160 / 172); beside many results 80 KB (100 queries: 73 / 67 / 68 / 74 / 80 / 80).
constexpr int MAX_STAGES = 6;

// The shared memory of a CTA: stages of a K chunk of rows (and of the queries); with a
// single query tile for several row tiles a CTA its queries stand behind the stages for
// good, as far as they leave half of the memory: loading the same few lines again for
// every row tile, from every SM at once, cost more than the rows themselves
// (922,893 rows of 42, 34 queries: 119 -> 40 us).
struct Ring {
  int stages, rows, bn;
  bool resident;
  __host__ __device__ int stage_bytes() const { return (rows + (resident ? 0 : bn)) * 128; }
  static Ring of(int rows, int bn, int chunks, bool many_rows) {
    Ring r{0, rows, bn, many_rows && chunks * bn * 128 <= RING_BYTES / 2};
    const int n = (RING_BYTES - (r.resident ? chunks * bn * 128 : 0)) / r.stage_bytes();
    const int most = (bn < 128 ? MAX_STAGES : MAX_STAGES - 1) * MMA_ROWS / rows;
    r.stages = n < most ? n : most;
    return r;
  }
};

// Bits of the waits that gave up, kept until circuit_op_int8_status reads them.
__device__ int g_error;

// Two results as the 16-bit values of one word.
__device__ __forceinline__ uint32_t two(__half, float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ uint32_t two(__nv_bfloat16, float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(h);
}

// W results of a lane's row, for queries `ld` bytes apart from `out` on.  `left` of
// them and live rows count.  16-bit results of full tiles go out as pairs of rows:
// neighbouring lanes swap one of every two columns, so that a warp store fills 64
// bytes of two queries.  Stores are marked as streaming, so that the results do not
// push the rows out of L2 (256 x 400,000 x 384 fp32: 114 -> 109 us).
template <typename T, int W>
__device__ __forceinline__ void store_columns(char* out, uint32_t ld, int64_t ld64, const uint32_t (&v)[W],
                                              const float* sq, float sr, float bias, bool live, int64_t left,
                                              bool pairs) {
  float s[W];
#pragma unroll
  for (int i = 0; i < W; i += 4) *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(sq + i);
  if constexpr (sizeof(T) == 2) {
    if (pairs && left >= W) {
      const bool odd = threadIdx.x & 1;
      const uint32_t pick = odd ? 0x3276u : 0x5410u;
      char* o = out + (odd ? (int64_t)ld - 2 : 0);
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const uint32_t mine = two(T{}, result((int)v[i], s[i], sr, bias), result((int)v[i + 1], s[i + 1], sr, bias));
        // even lanes keep column i of both rows, odd lanes column i + 1
        const uint32_t other = __shfl_xor_sync(FULL_MASK, mine, 1);
        __stcs(reinterpret_cast<uint32_t*>(o + (uint64_t)ld * (uint32_t)i), __byte_perm(mine, other, pick));
      }
      return;
    }
  }
  if (!live) return;
  if (left >= W && ld) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      __stcs(reinterpret_cast<T*>(out + (uint64_t)ld * (uint32_t)i), RowType<T>::put(result((int)v[i], s[i], sr, bias)));
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) *reinterpret_cast<T*>(out + ld64 * i) = RowType<T>::put(result((int)v[i], s[i], sr, bias));
  }
}

// An epilogue warp's loop over its group's units: 32 rows of the tile (its TMEM
// lanes) from row_off on, COLS columns.  The next unit's scales and the next 16
// columns are on their way while the present ones are stored.  Once a wait has given
// up, the results that it would have brought are NaN.
template <typename T, int BN, int SUBS, typename Release>
__device__ __forceinline__ bool epilogue(const ScoresParams& P, uint32_t tmem, float* sq, Units un, int64_t units,
                                         int tile_rows, int row_off, uint64_t* acc_full, Release release) {
  constexpr int PARTS = column_parts(BN), GROUPS = tile_groups(BN) / SUBS, NB = accumulators(BN, SUBS), COLS = BN / PARTS;
  constexpr int W = 16, N = COLS / W, SQ = (COLS + 31) / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3;
  const int part = (warp >> 2) % PARTS, sub = (warp >> 2) / PARTS % SUBS, group = (warp >> 2) / PARTS / SUBS;
  const uint32_t taddr = tmem + ((uint32_t)(32 * quarter) << 16) + (uint32_t)(sub * BN + part * COLS);
  const int64_t ld64 = P.out_stride * (int64_t)sizeof(T);
  const uint32_t ld = ld64 < (1ll << 32) ? (uint32_t)ld64 : 0u;
  float sr = 0.f, bias = 0.f, sqv[SQ];
  int64_t row0 = 0, q0 = 0;
  auto fetch = [&]() {  // of unit un
    row0 = un.rt * tile_rows + row_off + sub * MMA_ROWS + 32 * quarter;
    q0 = (int64_t)un.qt * BN + part * COLS;
    const bool live = row0 + lane < P.n;
    sr = live ? P.scales[row0 + lane] : 0.f;
    bias = live && P.bias ? P.bias[row0 + lane] : 0.f;
#pragma unroll
    for (int i = 0; i < SQ; ++i)
      sqv[i] = 32 * i + lane < COLS && q0 + 32 * i + lane < P.nq ? P.q_scales[q0 + 32 * i + lane] : 0.f;
  };
  for (int i = 0; i < group; ++i) un.next();
  if (un.u < units) fetch();
  bool ok = true;
  for (int it = group; un.u < units; it += GROUPS) {
    const int b = it % NB;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < SQ; ++i)
      if (32 * i + lane < COLS) sq[32 * i + lane] = sqv[i];
    __syncwarp();
    const int64_t row = row0 + lane, left = P.nq - q0;
    const bool pairs = P.pairs && ld && row0 + 32 <= P.n;
    char* out = reinterpret_cast<char*>(P.out) + q0 * ld64 + row * (int64_t)sizeof(T);
    float s = sr;
    const float bb = bias;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) un.next();
    if (un.u < units) fetch();
    ok = ok && __all_sync(FULL_MASK, mbar_wait(&acc_full[b], (uint32_t)(it / NB) & 1u, &g_error, ERR_TIMEOUT_FULL));
    if (!ok) s = __uint_as_float(0x7fffffffu);
    tc::fence_after();
    uint32_t v[2][W];
    tc::ld_32x32b_x16(taddr + (uint32_t)(b * BN * SUBS), v[0]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      tc::wait_ld();
      if (i + 1 < N) {
        tc::ld_32x32b_x16(taddr + (uint32_t)(b * BN * SUBS + (i + 1) * W), v[(i + 1) & 1]);
      } else {
        tc::fence_before();
        __syncwarp();
        if (lane == 0) release(b);
      }
      if (i * W < left)
        store_columns<T, W>(out + i * W * ld64, ld, ld64, v[i & 1], sq + i * W, s, bb, row < P.n, left - i * W, pairs);
    }
  }
  return ok;
}

template <typename T, int BN, int SUBS>
__global__ void __launch_bounds__(MMA_THREADS, 1)
    k_scores_mma(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap cmap, ScoresParams P,
                 int q_tiles, int64_t units, Ring ring) {
  constexpr int EW = EPILOGUE_WARPS, NB = accumulators(BN, SUBS), TILE = MMA_ROWS * SUBS;
  const int S = ring.stages, STAGE = ring.stage_bytes();
  extern __shared__ __align__(128) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[NB], acc_empty[NB], q_full;
  __shared__ uint32_t tmem_base;
  __shared__ int s_failed;
  __shared__ __align__(16) float s_sq[EW][BN / column_parts(BN)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = (P.d + 127) >> 7;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4 * column_parts(BN) * SUBS);  // one lane of each epilogue warp of a unit
    }
    mbar_init(&q_full, 1);
    s_failed = 0;
    fence_mbar_init();
  }
  if (threadIdx.x == 32 * EW) {
    tc::prefetch_map(&cmap);
    tc::prefetch_map(&qmap);
  }
  if (warp == EW + 1) tc::tmem_alloc(&tmem_base, NB * BN * SUBS);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_base;
  griddep_wait();  // codes and scales may come from the kernel before
  griddep_launch();

  if (warp == EW) {
    if (lane == 0) {
      int s = 0;
      int64_t filled = 0;
      uint32_t ph = 0;
      bool ok = true;
      if (ring.resident) {
        mbar_arrive_expect_tx(&q_full, (uint32_t)(chunks * BN * 128));
        for (int j = 0; j < chunks; ++j) tc::tma_load_2d(smem + S * STAGE + j * BN * 128, &qmap, 128 * j, 0, &q_full);
      }
      for (Units un(blockIdx.x, gridDim.x, q_tiles); un.u < units && ok; un.next()) {
        const int row0 = (int)(un.rt * TILE), q0 = un.qt * BN;
        for (int j = 0; j < chunks; ++j, ++filled) {
          if (filled >= S && !mbar_wait(&empty[s], ph ^ 1u, &g_error, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          mbar_arrive_expect_tx(&full[s], STAGE);  // out-of-range rows and columns arrive as zeros
          unsigned char* dst = smem + s * STAGE;
          tc::tma_load_2d(dst, &cmap, 128 * j, row0, &full[s]);
          if (!ring.resident) tc::tma_load_2d(dst + TILE * 128, &qmap, 128 * j, q0, &full[s]);
          if (++s == S) { s = 0; ph ^= 1u; }
        }
      }
      // the last commits to the empty barriers have landed before this CTA exits
      for (int64_t t = filled > S ? filled - S : 0; t < filled && ok; ++t)
        ok = mbar_wait(&empty[t % S], (uint32_t)(t / S) & 1u, &g_error, ERR_TIMEOUT_EMPTY);
      if (!ok) s_failed = 1;
    }
  } else if (warp == EW + 1) {
    constexpr uint32_t idesc = tc::idesc_s8(MMA_ROWS, BN);
    const uint32_t sbase = smem_u32(smem);
    // the chunk's queries: beside its rows in the stage, or chunk by chunk behind the ring
    const uint64_t dA = tc::sdesc_k_sw128(sbase),
                   dB = tc::sdesc_k_sw128(sbase + (ring.resident ? S * STAGE : TILE * 128));
    const int tail = (P.d - (chunks - 1) * 128 + 31) >> 5;  // K steps of 32 in the last chunk
    int s = 0, it = 0;
    uint32_t ph = 0;
    bool ok = !ring.resident || __all_sync(FULL_MASK, mbar_wait(&q_full, 0u, &g_error, ERR_TIMEOUT_FULL));
    for (int64_t u = blockIdx.x; u < units && ok; u += gridDim.x, ++it) {
      const int b = it % NB;
      if (it >= NB && !__all_sync(FULL_MASK, mbar_wait(&acc_empty[b], (uint32_t)(it / NB - 1) & 1u, &g_error,
                                                      ERR_TIMEOUT_EMPTY))) {
        ok = false;
        break;
      }
      tc::fence_after();
      const uint32_t acc = tmem + (uint32_t)(b * BN * SUBS);
      for (int j = 0; j < chunks; ++j) {
        if (!__all_sync(FULL_MASK, mbar_wait(&full[s], ph, &g_error, ERR_TIMEOUT_FULL))) { ok = false; break; }
        tc::fence_after();
        if (tc::elect_one()) {
          const uint64_t a = dA + ((uint32_t)(s * STAGE) >> 4);
          const uint64_t q = dB + ((uint32_t)(ring.resident ? j * BN * 128 : s * STAGE) >> 4);
          const int steps = j + 1 < chunks ? 4 : tail;
#pragma unroll
          for (int sub = 0; sub < SUBS; ++sub)
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 32 bytes of K further: 2 units of 16 bytes
              if (k < steps)
                tc::mma_s8_ss(acc + (uint32_t)(sub * BN), a + sub * (MMA_ROWS * 128 >> 4) + 2 * k, q + 2 * k, idesc,
                              (j | k) != 0 ? 1u : 0u);
          tc::commit(&empty[s]);
        }
        __syncwarp();
        if (++s == S) { s = 0; ph ^= 1u; }
      }
      if (ok && tc::elect_one()) tc::commit(&acc_full[b]);
      __syncwarp();
    }
    if (!ok && lane == 0) s_failed = 1;
  } else {
    const bool ok = epilogue<T, BN, SUBS>(P, tmem, s_sq[warp], Units(blockIdx.x, gridDim.x, q_tiles), units, TILE, 0,
                                          acc_full, [&](int b) { mbar_arrive(&acc_empty[b]); });
    if (!ok && lane == 0) s_failed = 1;
  }
  tc::fence_before();
  __syncthreads();
  if (s_failed) grace_period();  // copies and MMAs of the failed waits end before the memory is freed
  if (warp == EW + 1) tc::tmem_dealloc(tmem, NB * BN * SUBS);
}

// The same for many queries with a CTA pair a unit of 256 rows x 256 queries: each
// CTA loads 128 rows and 128 queries of a chunk (32 KB against the 48 KB of a
// single CTA's 128 x 256 tile, and the operands' way from L2 is what bounds the
// single CTA), the even CTA issues MMAs over both CTAs' shared memory, and each
// CTA's TMEM holds its 128 rows against all 256 queries.
constexpr int PAIR_BN = 256;
constexpr int PAIR_STAGE = (MMA_ROWS + PAIR_BN / 2) * 128;
constexpr int PAIR_STAGES = RING_BYTES / PAIR_STAGE;

template <typename T>
__global__ void __launch_bounds__(MMA_THREADS, 1)
    k_scores_pair(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap cmap, ScoresParams P,
                  int q_tiles, int64_t units, int S) {
  constexpr int EW = EPILOGUE_WARPS;
  static_assert(accumulators(PAIR_BN) == 2 && tile_groups(PAIR_BN) == 1, "two accumulators, every warp on every tile");
  extern __shared__ __align__(128) unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  // full and acc_empty are used in the even CTA only, empty and acc_full in both
  __shared__ uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int s_failed;
  __shared__ __align__(16) float s_sq[EW][PAIR_BN / column_parts(PAIR_BN)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = (P.d + 127) >> 7;
  const uint32_t rank = tc::cluster_ctarank();
  const int64_t first = blockIdx.x >> 1, step = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * EW);  // one lane of each epilogue warp of both CTAs
    }
    s_failed = 0;
    tc::fence_mbar_init_cluster();
    fence_mbar_init();
  }
  if (threadIdx.x == 32 * EW) {
    tc::prefetch_map(&cmap);
    tc::prefetch_map(&qmap);
  }
  if (warp == EW + 1) tc::tmem_alloc_pair(&tmem_base, 2 * PAIR_BN);
  tc::fence_before();
  tc::cluster_sync();  // barriers and the pair's TMEM exist before any remote access
  tc::fence_after();
  const uint32_t tmem = tmem_base;
  griddep_wait();  // codes and scales may come from the kernel before
  griddep_launch();
  const uint32_t lead_full = tc::mapa_shared(smem_u32(&full[0]), 0);
  const uint32_t lead_acc_empty = tc::mapa_shared(smem_u32(&acc_empty[0]), 0);

  if (warp == EW) {
    if (lane == 0) {
      int s = 0;
      int64_t filled = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (Units un(first, step, q_tiles); un.u < units && ok; un.next()) {
        const int row0 = (int)(un.rt * 2 * MMA_ROWS + rank * MMA_ROWS);
        const int q0 = un.qt * PAIR_BN + (int)rank * (PAIR_BN / 2);
        for (int j = 0; j < chunks; ++j, ++filled) {
          if (filled >= S && !mbar_wait(&empty[s], ph ^ 1u, &g_error, ERR_TIMEOUT_EMPTY)) { ok = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * PAIR_STAGE);  // both CTAs' copies
          unsigned char* dst = smem + s * PAIR_STAGE;
          const uint32_t bar = lead_full + 8u * (uint32_t)s;
          tc::tma_load_2d_pair(dst, &cmap, 128 * j, row0, bar);
          tc::tma_load_2d_pair(dst + MMA_ROWS * 128, &qmap, 128 * j, q0, bar);
          if (++s == S) { s = 0; ph ^= 1u; }
        }
      }
      for (int64_t t = filled > S ? filled - S : 0; t < filled && ok; ++t)
        ok = mbar_wait(&empty[t % S], (uint32_t)(t / S) & 1u, &g_error, ERR_TIMEOUT_EMPTY);
      if (!ok) s_failed = 1;
    }
  } else if (warp == EW + 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = tc::idesc_s8(2 * MMA_ROWS, PAIR_BN);
      const uint32_t sbase = smem_u32(smem);
      const uint64_t dA = tc::sdesc_k_sw128(sbase), dB = tc::sdesc_k_sw128(sbase + MMA_ROWS * 128);
      const uint32_t empty0 = tc::mapa_shared(smem_u32(&empty[0]), 0), empty1 = tc::mapa_shared(smem_u32(&empty[0]), 1);
      const uint32_t accf0 = tc::mapa_shared(smem_u32(&acc_full[0]), 0);
      const uint32_t accf1 = tc::mapa_shared(smem_u32(&acc_full[0]), 1);
      const int tail = (P.d - (chunks - 1) * 128 + 31) >> 5;
      int s = 0, it = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int64_t u = first; u < units && ok; u += step, ++it) {
        const int b = it & 1;
        if (it >= 2 && !__all_sync(FULL_MASK, tc::mbar_wait_cluster(&acc_empty[b], (uint32_t)(it / 2 - 1) & 1u, &g_error,
                                                                    ERR_TIMEOUT_EMPTY))) {
          ok = false;
          break;
        }
        tc::fence_after();
        const uint32_t acc = tmem + (uint32_t)(b * PAIR_BN);
        for (int j = 0; j < chunks; ++j) {
          if (!__all_sync(FULL_MASK, mbar_wait(&full[s], ph, &g_error, ERR_TIMEOUT_FULL))) { ok = false; break; }
          tc::fence_after();
          if (tc::elect_one()) {
            const uint64_t off = (uint64_t)((uint32_t)(s * PAIR_STAGE) >> 4);
            const int steps = j + 1 < chunks ? 4 : tail;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (k < steps) tc::mma_s8_ss_pair(acc, dA + off + 2 * k, dB + off + 2 * k, idesc, (j | k) != 0 ? 1u : 0u);
            tc::commit_pair(empty0 + 8u * (uint32_t)s);
            tc::commit_pair(empty1 + 8u * (uint32_t)s);
          }
          __syncwarp();
          if (++s == S) { s = 0; ph ^= 1u; }
        }
        if (ok && tc::elect_one()) {
          tc::commit_pair(accf0 + 8u * (uint32_t)b);
          tc::commit_pair(accf1 + 8u * (uint32_t)b);
        }
        __syncwarp();
      }
      if (!ok && lane == 0) s_failed = 1;
    }
  } else {
    const bool ok = epilogue<T, PAIR_BN, 1>(P, tmem, s_sq[warp], Units(first, step, q_tiles), units, 2 * MMA_ROWS,
                                      (int)rank * MMA_ROWS, acc_full,
                                      [&](int b) { tc::mbar_arrive_remote(lead_acc_empty + 8u * (uint32_t)b); });
    if (!ok && lane == 0) s_failed = 1;
  }
  tc::fence_before();
  __syncthreads();
  if (s_failed) grace_period();  // copies and MMAs of the failed waits end before the memory is freed
  tc::cluster_sync();  // neither CTA leaves while the other may still arrive on its barriers
  if (warp == EW + 1) tc::tmem_dealloc_pair(tmem, 2 * PAIR_BN);
}

static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ok ? p : nullptr);
  }();
  return fn;
}
// [rows, d] codes as boxes of box_rows rows x 128 bytes, 128-byte swizzle.
static bool code_map(CUtensorMap* map, const int8_t* base, int64_t rows, int d, int64_t stride, int box_rows) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)stride};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
static int sm_count() {
  static std::atomic<int> known[SmemOptIn::kMaxDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= SmemOptIn::kMaxDevices) return 148;
  if ((n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, int BN, int SUBS>
static int launch_mma_units(const ScoresParams& P, cudaStream_t st) {
  constexpr int rows = MMA_ROWS * SUBS;
  CUtensorMap qmap, cmap;
  if (!code_map(&qmap, P.q, P.nq, P.d, P.q_stride, BN) || !code_map(&cmap, P.codes, P.n, P.d, P.code_stride, rows))
    return bad("int8_scores: cuTensorMapEncodeTiled refused the code rows");
  constexpr int smem = RING_BYTES + 1024;
  static SmemOptIn opt_in;
  const int rc = check(opt_in.ensure(reinterpret_cast<const void*>(k_scores_mma<T, BN, SUBS>), smem),
                       "int8_scores shared memory");
  if (rc) return rc;
  const int q_tiles = (int)((P.nq + BN - 1) / BN);
  const int64_t units = (P.n + rows - 1) / rows * q_tiles, sms = sm_count();
  return check(launch(k_scores_mma<T, BN, SUBS>, dim3((unsigned)(units < sms ? units : sms)), MMA_THREADS, smem, 1, st,
                      qmap, cmap, P, q_tiles, units,
                      Ring::of(rows, BN, (P.d + 127) / 128, q_tiles == 1 && units > 2 * sms)),
               "int8_scores launch");
}
template <typename T, int BN>
static int launch_mma(const ScoresParams& P, cudaStream_t st) {
  // two tiles a unit: rows of one chunk, several units an SM
  if constexpr (BN <= 64) {
    if (P.d <= 128 && P.n > 4 * 2 * MMA_ROWS * (int64_t)sm_count()) return launch_mma_units<T, BN, 2>(P, st);
  }
  return launch_mma_units<T, BN, 1>(P, st);
}

template <typename T, int NQ>
static int launch_rows(const ScoresParams& P, cudaStream_t st) {
  static_assert(NQ * CIRCUIT_INT8_MAX_DIM <= 48 * 1024, "the queries fit the default shared memory");
  const int smem = NQ * ((P.d + 15) / 16) * 16;
  const int64_t blocks = (P.n + 31) / 32;
  const dim3 grid((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), (unsigned)((P.nq + NQ - 1) / NQ));
  return check(launch(k_scores_rows<T, NQ>, grid, 256, smem, 1, st, P), "int8_scores launch");
}
template <typename T>
static int launch_pair(const ScoresParams& P, cudaStream_t st) {
  CUtensorMap qmap, cmap;
  if (!code_map(&qmap, P.q, P.nq, P.d, P.q_stride, PAIR_BN / 2) ||
      !code_map(&cmap, P.codes, P.n, P.d, P.code_stride, MMA_ROWS))
    return bad("int8_scores: cuTensorMapEncodeTiled refused the code rows");
  constexpr int smem = PAIR_STAGES * PAIR_STAGE + 1024;
  static SmemOptIn opt_in;
  const int rc = check(opt_in.ensure(reinterpret_cast<const void*>(k_scores_pair<T>), smem), "int8_scores shared memory");
  if (rc) return rc;
  const int q_tiles = (int)((P.nq + PAIR_BN - 1) / PAIR_BN);
  const int64_t units = (P.n + 2 * MMA_ROWS - 1) / (2 * MMA_ROWS) * q_tiles, pairs = sm_count() / 2;
  // short sums are bound by the results' way out, which less in flight disturbs less (200,000 x 100 fp16, 558 queries: 4
  // stages 63 us, 6 stages 69; 1,024 x 40,000 x 768: 34 and 31)
  const int stages = P.d <= 512 ? 4 : PAIR_STAGES;
  return check(launch(k_scores_pair<T>, dim3((unsigned)(2 * (units < pairs ? units : pairs))), MMA_THREADS, smem, 2, st, qmap,
                      cmap, P, q_tiles, units, stages),
               "int8_scores launch");
}

template <typename T>
static int scores(const ScoresParams& P, cudaStream_t st) {
  // One or two queries on few bytes: the row kernel starts faster (5,183 x 384: 3.0 against 3.6 us, 4,096 x 2,048: 5.5
  // against 7.1); from 16 MB on the ring of bulk copies keeps more in flight (50,000 x 384: 5.8 and 5.9 us,
  // 2,000,000 x 384: 223 against 127).
  if (P.nq <= 2 && P.n * P.d <= (16 << 20))
    return P.nq == 1 ? launch_rows<T, 1>(P, st) : launch_rows<T, 2>(P, st);
  if (P.nq <= 16) return launch_mma<T, 16>(P, st);
  if (P.nq <= 32) return launch_mma<T, 32>(P, st);
  if (P.nq <= 64) return launch_mma<T, 64>(P, st);
  if (P.nq <= 128) return launch_mma<T, 128>(P, st);
  // Pairs of CTAs take 256 x 256 tiles, single ones 128 x 128: a round of pairs costs about one and a half rounds of
  // single CTAs and does twice as much, when it is full (300 queries against 50,000 rows of 384: 6 rounds 22.6 us, 8
  // single ones 16.5; 1,024 against 40,000 of 768: 9 rounds 31.8 us, 17 single ones 42.6).
  const int64_t sms = sm_count(), pairs = sms / 2 > 0 ? sms / 2 : 1;
  const int64_t single = ((P.n + 127) / 128 * ((P.nq + 127) / 128) + sms - 1) / sms;
  const int64_t paired = ((P.n + 255) / 256 * ((P.nq + 255) / 256) + pairs - 1) / pairs;
  if (2 * single < 3 * paired) return launch_mma<T, 128>(P, st);
  return launch_pair<T>(P, st);
}

}  // namespace i8
}  // namespace cb

using namespace cb::i8;

extern "C" {

int circuit_op_int8_scores(const int8_t* queries, int64_t query_stride, const float* query_scales, int64_t num_queries,
                           const int8_t* codes, int64_t code_stride, const float* scales, int64_t n, int dim,
                           const float* bias, void* out, int dtype, int64_t out_stride, void* stream) {
  const int e = type_bytes(dtype);
  if (!e) return bad("int8_scores: dtype must be CIRCUIT_F32, CIRCUIT_F16 or CIRCUIT_BF16");
  if (dim < 1 || dim > CIRCUIT_INT8_MAX_DIM) return bad("int8_scores: dim must be in [1, 16384]");
  if (num_queries < 0 || num_queries > CIRCUIT_INT8_MAX_QUERIES)
    return bad("int8_scores: the number of queries must be in [0, 65535]");
  if (n < 0 || n > 0x7fffffffLL) return bad("int8_scores: n must be in [0, 2^31)");
  if (num_queries == 0 || n == 0) return CIRCUIT_OK;
  if (!queries || !query_scales || !codes || !scales || !out) return bad("int8_scores: null pointer");
  const int64_t padded = (dim + 15) / 16 * 16;
  if (query_stride < padded || code_stride < padded || !on16(queries, query_stride) || !on16(codes, code_stride))
    return bad("int8_scores: code rows must start on 16 bytes and be padded to a multiple of 16");
  if (out_stride < n) return bad("int8_scores: out_stride is smaller than n");
  if ((uintptr_t)out % e || ((uintptr_t)query_scales | (uintptr_t)scales | (uintptr_t)bias) % 4)
    return bad("int8_scores: a pointer is not aligned to its type");
  const ScoresParams P{queries, query_scales, codes, scales, bias, out, num_queries, n, query_stride, code_stride,
                       out_stride, dim,
                       e == 2 && ((uintptr_t)out & 3) == 0 && out_stride % 2 == 0};
  cudaStream_t st = (cudaStream_t)stream;
  int rc = CIRCUIT_ERR_CUDA;
  try {
    rc = dtype == CIRCUIT_F32   ? scores<float>(P, st)
         : dtype == CIRCUIT_F16 ? scores<__half>(P, st)
                                : scores<__nv_bfloat16>(P, st);
  } catch (...) {  // a lock of the host's that failed
    return bad("int8_scores: the host ran out of a resource");
  }
  return rc ? rc : check(cudaGetLastError(), "int8_scores launch");
}

int circuit_op_int8_status(void* stream) {
  cudaStream_t st = (cudaStream_t)stream;  // copies on it too: others would wait for the work of every stream
  int bits = 0;
  const int none = 0;
  int rc = check(cudaMemcpyFromSymbolAsync(&bits, g_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st), "int8_status");
  if (!rc) rc = check(cudaStreamSynchronize(st), "int8_status");
  if (!rc && bits) {
    rc = check(cudaMemcpyToSymbolAsync(g_error, &none, sizeof(int), 0, cudaMemcpyHostToDevice, st), "int8_status");
    if (!rc) rc = check(cudaStreamSynchronize(st), "int8_status");
  }
  if (rc || !bits) return rc;
  bad("int8_scores: a bounded wait on the device gave up; its results are NaN");
  return CIRCUIT_ERR_TIMEOUT;
}

}  // extern "C"
