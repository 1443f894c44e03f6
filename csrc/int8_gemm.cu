// Products of 8-bit integers on tcgen05 (kind::i8), weights as the MMA's rows: out[row, feature] = sx[row] sw[feature] qx[row] · qw[feature].
//
// 128 weight rows fill the MMA's lanes, up to 256 rows of activations its N; a TMA ring of 128-byte k-blocks (128 values), one thread issues the MMAs, int32 sums in
// TMEM, two accumulators.  Sums leave through shared memory as [row][feature], so that a thread finishes four neighbouring features of a row: both scales, the
// residual or the gate, one rounding.  One matrix, or one per expert: rows come ordered by expert, at any row, no padding between experts; a tile of rows that runs
// past its expert's end computes rows of the next one and does not store them.
// The launch ahead is always the one that brings the activations to 8 bits, which lets this one start when the kernels before it are done (or, with resident weights, at
// once): offsets and weights are read without waiting for it.
// Bound by the weights' way from memory with few rows: one B200, us in a chain of cold weights, the rows' kernel included, 1 x 28672 x 4096 20.1 (5.9 TB/s), 16 x 4096 x 4096 7.8, 48 x
// 28672 x 4096 gated 22.4 (5.4 TB/s), 64 tokens x 4 of 32 experts of 2048 x 1024 12.9 (5.3 TB/s); with more by the operands' way from L2 (24 KB for 128 x 64 x 128).
// Few tiles: the CTAs of a cluster share one and take a part of K each; the partials meet in distributed shared memory, whole numbers, so their order
// changes nothing.
#include <type_traits>

#include "int8.cuh"
#include "jllama_b200.h"
#include "tcgen05.cuh"

namespace jl {

constexpr int I8S_BM = 128, I8S_BK = 128, I8S_THREADS = 256;      // warp 0: TMA, warp 1: MMA, warp 2: TMEM; 4-7 (split: all): results
constexpr uint32_t I8S_A_BYTES = I8S_BM * I8S_BK, I8S_STAGING = 16 * I8S_BM * 4;
constexpr int I8S_PARTS = 8;                                      // of K, at most
constexpr int I8S_HALF = 112 * 1024, I8S_WIDE = 201 * 1024;       // shared memory of a CTA: of two an SM, of one

struct Int8Swap {
  Int8Out o;
  Int8Work work;
  int K, nb, stages, ksplit;        // rows of a tile: nb, a multiple of 16
  uint32_t cols, idesc;
};

__device__ __forceinline__ uint32_t i8s_mapa(uint32_t local_addr, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local_addr), "r"(rank));
  return a;
}
__device__ __forceinline__ int4 i8s_ld_cluster(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int MODE, bool SPLIT, int KIND>
__global__ void __launch_bounds__(I8S_THREADS, 2)
int8_swap_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Int8Swap p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  const int stages = p.stages, ksplit = SPLIT ? p.ksplit : 1;
  const uint32_t b_bytes = (uint32_t)p.nb * I8S_BK, stage_bytes = I8S_A_BYTES + b_bytes;
  const uint32_t staging = smem_base + stages * stage_bytes;    // !SPLIT: 16 rows x 32 features for each epilogue warp
  const uint32_t bars = staging + (SPLIT ? 0u : I8S_STAGING);   // full[stages] | empty[stages] | tfull[2] | tempty[2]
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
  auto tfull_bar = [&](int s) { return bars + 8u * (2 * stages + s); };
  auto tempty_bar = [&](int s) { return bars + 8u * (2 * stages + 2 + s); };
  const uint32_t tmem_slot = bars + 8u * (2 * stages + 4);
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - tc::smem_u32(smem_raw)));
  int* table = reinterpret_cast<int*>(smem_raw + (tmem_slot + 16 - tc::smem_u32(smem_raw)));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_kb = (p.K + I8S_BK - 1) / I8S_BK;
  const int tile0 = (int)blockIdx.x / ksplit, tstep = (int)gridDim.x / ksplit;      // SPLIT: one tile, its parts are the CTAs of a cluster
  const int rank = (int)blockIdx.x % ksplit, kb0 = rank * num_kb / ksplit, kb1 = (rank + 1) * num_kb / ksplit;

  if (warp == 0 && lane == 0) {
    tc::prefetch_tensormap(&tmap_w);
    tc::prefetch_tensormap(&tmap_x);
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < stages; ++s) { tc::mbar_init(full_bar(s), 1); tc::mbar_init(empty_bar(s), 1); }
    for (int s = 0; s < 2; ++s) { tc::mbar_init(tfull_bar(s), 1); tc::mbar_init(tempty_bar(s), 4); }
    tc::fence_barrier_init();
  }
  if (warp == 2) tc::tmem_alloc(tmem_slot, SPLIT ? p.cols : 2 * p.cols);
  if (warp == 3) {
    i8_list(p.work, table);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_ptr;
  pdl_launch_dependents();
  const int tiles = table[p.work.experts];

  if (warp == 0) {
    // ===================================================== TMA producer
    if (lane == 0) {
      int pre = 0;
      if (tile0 < tiles) {                                      // weights do not wait for the activations
        Int8Walk walk;
        const Int8Tile t = walk.at(p.work, table, tile0);
        pre = kb1 - kb0 < stages ? kb1 - kb0 : stages;
        for (int i = 0; i < pre; ++i) {
          tc::mbar_expect_tx(full_bar(i), stage_bytes);
          tc::tma_load_2d(smem_base + i * stage_bytes, &tmap_w, full_bar(i), (kb0 + i) * I8S_BK, t.expert * p.o.N + t.col * I8S_BM, tc::EVICT_FIRST);
        }
      }
      pdl_wait();
      Int8Walk walk;
      int stage = 0; uint32_t phase = 0;
      for (int tile = tile0; tile < tiles; tile += tstep) {
        const Int8Tile t = walk.at(p.work, table, tile);
        const int w_row = t.expert * p.o.N + t.col * I8S_BM;
        for (int kb = kb0; kb < kb1; ++kb) {
          const uint32_t sa = smem_base + stage * stage_bytes;
          if (pre > 0) {
            --pre;
          } else {
            tc::mbar_wait(empty_bar(stage), phase ^ 1);
            tc::mbar_expect_tx(full_bar(stage), stage_bytes);
            tc::tma_load_2d(sa, &tmap_w, full_bar(stage), kb * I8S_BK, w_row, tc::EVICT_FIRST);
          }
          tc::tma_load_2d(sa + I8S_A_BYTES, &tmap_x, full_bar(stage), kb * I8S_BK, t.row0, tc::EVICT_LAST);
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ===================================================== MMA issuer (single thread)
    if (lane == 0) {
      int stage = 0, it = 0; uint32_t phase = 0;
      for (int tile = tile0; tile < tiles; tile += tstep, ++it) {
        const int as = it & 1;
        if constexpr (!SPLIT) {
          tc::mbar_wait(tempty_bar(as), ((it >> 1) & 1) ^ 1);      // the epilogue has drained this accumulator
          tc::fence_after_sync();
        }
        const uint32_t d = tmem_base + as * p.cols;
        for (int kb = kb0; kb < kb1; ++kb) {
          tc::mbar_wait(full_bar(stage), phase);
          tc::fence_after_sync();
          const uint32_t sa = smem_base + stage * stage_bytes;
          const uint64_t da = tc::smem_desc_kmajor_sw128(sa), db = tc::smem_desc_kmajor_sw128(sa + I8S_A_BYTES);
#pragma unroll
          for (int k = 0; k < I8S_BK / 32; ++k)             // +32 bytes per UMMA_K inside the swizzle span
            tc::mma_ss_i8(d, da + 2 * k, db + 2 * k, p.idesc, kb != kb0 || k != 0);
          tc::mma_commit(empty_bar(stage));                 // frees the smem slot when these MMAs retire
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
        tc::mma_commit(tfull_bar(as));
      }
    }
    __syncwarp();
  }

  // TMEM lane = weight row, column = row of activations
  const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
  auto to_shared = [&](uint32_t t_col, uint32_t at, int pitch) {      // 16 rows
    uint32_t v[16];
    tc::tmem_ld16(t_col, v);
    tc::tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + j * pitch), "r"(v[j]) : "memory");
  };
  auto feature_scales = [&](int expert, int f0, float (&sw)[4]) {
    const float* s = p.o.ws + (size_t)expert * p.o.N + f0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sw[i] = f0 + i < p.o.N ? s[i] : 0.0f;
  };
  constexpr int DEPTH = KIND == DT_F32 ? 1 : 2;             // how far ahead residuals are asked for: 32 registers
  if constexpr (!SPLIT) {
    // ===================================================== epilogue of a persistent CTA: warps 4-7, 16 rows at a time
    if (warp >= 4) {
      pdl_wait();                                           // scales, residual, output: after the previous kernel
      const uint32_t st = staging + (warp & 3) * (I8S_STAGING / 4);
      Int8Walk walk;
      int it = 0;
      for (int tile = tile0; tile < tiles; tile += tstep, ++it) {
        const Int8Tile t = walk.at(p.work, table, tile);
        const int as = it & 1, f0 = t.col * I8S_BM + (warp & 3) * 32 + 4 * (lane & 7);
        float sw[4], sx[2];                                 // features'; rows' of two times 32, a lane each
        feature_scales(t.expert, f0, sw);
        auto row_scales = [&](int c) {
#pragma unroll
          for (int i = 0; i < 2; ++i) sx[i] = c + 32 * i + lane < t.rows ? p.o.xs[t.row0 + c + 32 * i + lane] : 0.0f;
        };
        row_scales(0);
        Int8Four<KIND> r4[DEPTH + 1][4];                    // residuals of 16 rows each, asked for while those before them are finished
        auto residuals = [&](int c, Int8Four<KIND>(&r)[4]) {
          if constexpr (MODE == I8_RESIDUAL) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (c + (lane >> 3) + 4 * u < t.rows) r[u].load(p.o, t.row0 + c + (lane >> 3) + 4 * u, f0);
          }
        };
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) residuals(16 * d, r4[d + 1]);
        tc::mbar_wait(tfull_bar(as), (it >> 1) & 1);
        tc::fence_after_sync();
        for (int c64 = 0; c64 < t.rows; c64 += 64) {
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
            const int c0 = c64 + 16 * q;
            if (c0 >= t.rows) break;
            to_shared(t_lane + as * p.cols + c0, st + lane * 4, 128);
            tc::fence_before_sync();
            __syncwarp();
            if (c0 + 16 >= t.rows && lane == 0) tc::mbar_arrive(tempty_bar(as));      // read: the sums of the tile after next may begin
#pragma unroll
            for (int d = 0; d < DEPTH; ++d)
#pragma unroll
              for (int u = 0; u < 4; ++u) r4[d][u] = r4[d + 1][u];
            residuals(c0 + 16 * DEPTH, r4[DEPTH]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int r = (lane >> 3) + 4 * u, row = c0 + r;
              const float s = __shfl_sync(0xffffffffu, q < 2 ? sx[0] : sx[1], 16 * (q & 1) + r);
              if (f0 >= p.o.N || row >= t.rows) continue;
              int x[4];
              asm volatile("ld.shared.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(st + r * 128 + (lane & 7) * 16) : "memory");
              i8_finish4<MODE, KIND>(p.o, t.row0 + row, f0, x, s, sw, r4[0][u]);
            }
            __syncwarp();
          }
          if (c64 + 64 < t.rows) row_scales(c64 + 64);
        }
      }
    }
  } else {
    // ===================================================== all warps: partial sums meet in the cluster (one tile, or none)
    pdl_wait();
    Int8Walk walk;
    Int8Tile t{0, 0, 0, 0};
    if (tile0 < tiles) t = walk.at(p.work, table, tile0);
    const int f0 = t.col * I8S_BM + 4 * lane, row = I8S_BM * 4;
    const uint32_t put = smem_base + ((warp & 3) * 32 + lane) * 4, get = smem_base + lane * 16;
    float sw[4];
    feature_scales(t.expert, f0, sw);
    auto share = [&]() {
      if (tile0 < tiles) tc::mbar_wait(tfull_bar(0), 0);
      tc::fence_after_sync();
      // the ring is free (all MMAs done) and takes the partial
      for (int c0 = (warp >> 2) * 16; c0 < t.rows; c0 += 32) to_shared(t_lane + c0, put + c0 * row, row);
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    };
    const int per = (t.rows + ksplit - 1) / ksplit, t_lo = rank * per, t_hi = min(t_lo + per, t.rows);
    // a warp takes U rows at a time, all ranks' parts of them on their way together; the first rows' scales and residuals before the sums are there
    auto meet = [&](auto ranks, auto many) {
      constexpr int R = decltype(ranks)::value, U = decltype(many)::value;
      float sx[DEPTH][U];
      Int8Four<KIND> r4[DEPTH][U];
      auto ahead = [&](int r0, int d) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r0 + 8 * u >= t_hi) continue;
          sx[d][u] = p.o.xs[t.row0 + r0 + 8 * u];
          if constexpr (MODE == I8_RESIDUAL) r4[d][u].load(p.o, t.row0 + r0 + 8 * u, f0);
        }
      };
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) ahead(t_lo + warp + 8 * U * d, d);
      share();
      for (int r0 = t_lo + warp; r0 < t_hi; r0 += 8 * U) {
        int4 part[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = r0 + 8 * u;
          if (at >= t_hi) continue;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (r < ksplit) part[u][r] = i8s_ld_cluster(i8s_mapa(get, r) + at * row);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = r0 + 8 * u;
          if (at >= t_hi) continue;
          int x[4] = {0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (r < ksplit) { x[0] += part[u][r].x; x[1] += part[u][r].y; x[2] += part[u][r].z; x[3] += part[u][r].w; }
          if (f0 < p.o.N) i8_finish4<MODE, KIND>(p.o, t.row0 + at, f0, x, sx[0][u], sw, r4[0][u]);
        }
#pragma unroll
        for (int d = 0; d + 1 < DEPTH; ++d)
#pragma unroll
          for (int u = 0; u < U; ++u) { sx[d][u] = sx[d + 1][u]; r4[d][u] = r4[d + 1][u]; }
        ahead(r0 + 8 * U * DEPTH, DEPTH - 1);
      }
    };
    if (ksplit <= 4) meet(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
    else meet(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");      // no CTA leaves while its partial may still be read
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 2) tc::tmem_dealloc(tmem_base, SPLIT ? p.cols : 2 * p.cols);
}

static size_t i8s_smem(int stages, int nb, bool split, int experts) {
  return (size_t)stages * (I8S_A_BYTES + nb * I8S_BK) + (split ? 0 : I8S_STAGING) + 8 * (2 * stages + 4) + 16 + 4 * i8_table_ints(experts) + 1024;
}

// Parts of K, a cluster's CTAs, at most `most` of at least four k-blocks each, for `tiles` tiles in `slots` CTAs
static int i8s_parts(long long tiles, int num_kb, int most, int slots) {
  long long ks = slots / tiles;
  if (ks > most) ks = most;
  if (ks > num_kb / 4) ks = num_kb / 4;
  return ks > 1 ? (int)ks : 1;
}
// Two CTAs an SM: clusters find place for about 264 CTAs (48 tiles of 100 rows, K 4096: 5 parts 12.6 us, 6 parts 18.5; 32 tiles of 6 rows, K 14336: 2 parts 20.7, 4 15.2, 8 13.1)
static int i8s_slots(int num_sms) { return 2 * num_sms - 32; }

// How a product of M rows with one matrix is cut: pieces of rows, parts of K, and whether a CTA has an SM and its shared memory to itself.  pieces 0: the pairs' kernel.
//
// Up to 64 rows the weights' stream is all there is: one piece, K in up to eight parts, two CTAs an SM.  With more, a deeper ring for one CTA an SM and fewer, longer parts pay (the parts'
// meeting takes 20 ns a row, a k-block 1.4 ns a row beside its weights); then pieces of half the rows, where that leaves K in as many parts or K is short; few features take
// more and smaller pieces, to use the SMs at all.  us, one piece in eight or four parts -> as below: 72 x 4096 x 4096 10.4 -> 9.8; 100 x 4096 x 4096 11.8 -> 10.0; 128 x 4096 x
// 14336 20.5 -> 18.0; 128 x 8192 x 2048 12.0 -> 10.2; 100 x 1024 x 1024 7.6 -> 6.3; 200 x 2048 x 8192 15.4 -> 13.3; 256 x 4096 x 4096 14.5 -> 13.5; 256 x 1024 x 4096 12.3 -> 9.7;
// 256 x 6144 x 4096 16.8 -> 15.2; 512 x 1024 x 4096 14.2 -> 11.8.  One piece stays better for a long K: 256 x 4096 x 14336 23.1 and 25.6, 160 x 4096 x 4096 11.2 and 11.7; and two CTAs an SM
// up to 80 rows over many features: 72 x 6144 x 4096 10.9 and 11.4.
// Beyond 256 rows pieces of 128 as long as each can have an SM, whatever their number (us here | in pairs: 600 x 1024 x 4096 13.4 | 17.4; 1024 x 2048 x 4096 18.8 | 21.4; 4096 x 128 x
// 8192 24.3 | 38.7; 333 x 6144 x 4096 16.4 | 18.9; 500 x 4608 x 4096 17.7 | 18.7; 8192 x 128 x 2048 16.0 | 17.4; in fewer pieces, K in parts, 130 x 4096 x 4096 10.7 | 16.3, 512 x 4096 x 4096 17.2 | 18.3).
// Pairs otherwise: K short (200 x 1024 x 1024 9.3 | 6.9, 333 x 1000 x 960 9.0 | 7.3) or many tiles (256 x 28672 x 4096 45 | 32, 512 x 6144 x 4096 19.4 | 18.8).
struct Int8Cut { int pieces, parts, wide; };
static Int8Cut i8s_cut(int M, int N, int K, int num_sms) {
  const int cols = (N + I8S_BM - 1) / I8S_BM, kb = (K + I8S_BK - 1) / I8S_BK, both = i8s_slots(num_sms), one = num_sms - 20;
  const bool few = cols <= 10;
  if (M <= 64) return {1, i8s_parts(cols, kb, I8S_PARTS, both), 0};
  if (M <= 128) {
    if (few) {
      const int c = (M + 47) / 48;
      return {c, i8s_parts((long long)cols * c, kb, 6, one), 0};
    }
    if (cols <= one / 2 && (M > 80 || cols <= one / 3)) return {1, i8s_parts(cols, kb, cols <= one / 6 ? 6 : 4, one), 1};
    return {1, i8s_parts(cols, kb, I8S_PARTS, both), 0};
  }
  if (kb < 16) return {0, 0, 0};
  const long long tiles = (long long)cols * ((M + 127) / 128);      // of 128 x 128
  if (M > 512) return tiles <= num_sms ? Int8Cut{(M + 127) / 128, i8s_parts(tiles, kb, 4, one), 1} : Int8Cut{0, 0, 0};
  if (few) {
    const int c = (M + 111) / 112 < 4 ? (M + 111) / 112 : 4;
    return {c, i8s_parts((long long)cols * c, kb, 6, one), 1};
  }
  if (M > 256) {
    const int ks = i8s_parts(2ll * cols, kb, 4, one);
    if (ks > 1) return {2, ks, 1};
    return tiles <= num_sms ? Int8Cut{(M + 127) / 128, 1, 1} : Int8Cut{0, 0, 0};
  }
  if (cols <= one / 6 || (kb <= 48 && M > 176)) {
    const int ks = i8s_parts(2ll * cols, kb, 4, one);
    if (ks > 1) return {2, ks, 1};
    const int two = i8s_parts(2ll * cols, kb, 4, both);
    return two > 1 ? Int8Cut{2, two, 0} : Int8Cut{0, 0, 0};
  }
  const int ks = i8s_parts(cols, kb, 4, one);
  return ks > 1 ? Int8Cut{1, ks, 1} : Int8Cut{0, 0, 0};
}

template <int MODE, int KIND>
static int swap_launch(const void* xq, const void* wq, Int8Swap p, int ldx, int ldw, bool wide, int num_sms, cudaStream_t stream) {
  const int E = p.work.experts;
  p.work.cols = (p.o.N + I8S_BM - 1) / I8S_BM;
  p.work.chunk = p.nb;
  const int num_kb = (p.K + I8S_BK - 1) / I8S_BK;
  const long long most = p.work.cols * i8_pieces(p.work, p.nb);      // tiles, at most
  JL_CHECK_ARG(most < (1ll << 30), "int8 product: %lld tiles", most);
  const bool split = p.ksplit > 1;
  p.cols = p.nb <= 32 ? 32 : p.nb <= 64 ? 64 : p.nb <= 128 ? 128 : 256;
  p.idesc = tc::idesc_s8_s32(I8S_BM, p.nb);
  const int stage = (int)I8S_A_BYTES + p.nb * I8S_BK, room = 4 * i8_table_ints(E) + (split ? 0 : (int)I8S_STAGING);
  int stages = ((wide ? I8S_WIDE : I8S_HALF) - 2048 - room) / stage;      // (2 KB: barriers, alignment)
  if (stages > 10) stages = 10;
  const int slots = wide ? num_sms : 2 * num_sms;
  const long long blocks = split ? (num_kb + p.ksplit - 1) / p.ksplit : (most + slots - 1) / slots * num_kb;
  const int tile = split ? (p.nb * I8S_BM * 4 + stage - 1) / stage : 2;                    // a split's partial fits the ring
  if (stages > blocks) stages = (int)blocks;
  if (stages < tile) stages = tile;
  p.stages = stages;
  CUtensorMap tw, tx;
  int rc;
  if ((rc = make_tmap_2d_i8(&tw, wq, (uint64_t)p.o.N * E, p.K, ldw, I8S_BM))) return rc;
  if ((rc = make_tmap_2d_i8(&tx, xq, p.work.rows, p.K, ldx, p.nb))) return rc;
  const size_t smem = i8s_smem(stages, p.nb, split, E);
  auto kern = split ? int8_swap_kernel<MODE, true, KIND> : int8_swap_kernel<MODE, false, KIND>;
  JL_CUDA(split ? (i8_room<int8_swap_kernel<MODE, true, KIND>>()) : (i8_room<int8_swap_kernel<MODE, false, KIND>>()));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(split ? most * p.ksplit : most < slots ? most : slots));
  cfg.blockDim = dim3(I8S_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (pdl_enabled()) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (split) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = p.ksplit;
    attr[na].val.clusterDim.y = 1;
    attr[na++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  count_launch();
  JL_CUDA(cudaLaunchKernelEx(&cfg, kern, tw, tx, p));
  return JL_OK;
}

int int8_rows(const void* x, int dtype, int M, int K, long long ldx, const int* rows, int n, const void* gain, float eps, void* q, int ldq, float* s, int early,
              cudaStream_t stream);

bool int8_vec_takes(int rows, int N, int K);
int int8_vec(const void* x, int dtype, long long ldx, const void* gain, float eps, const void* wq, int ldw, Int8Out o, int rows, int K, int mode, bool early, int num_sms,
             cudaStream_t stream);
bool int8_vec_takes_pairs(int pairs, int N, int K);
bool int8_vec_holds_pairs(int pairs, int K);
int int8_vec_pairs(const void* x, int dtype, int M, long long ldx, const int* index, int pairs, const int* offsets, const int* choice, int top, int experts, const void* wq, int ldw, Int8Out o, int K, int mode,
                   int num_sms, cudaStream_t stream);
int int8_pair(const void* xq, int ldx, const void* wq, int ldw, Int8Out o, Int8Work work, int K, int mode, int num_sms, cudaStream_t stream);

// nb: rows of a tile; parts of K; wide: a CTA has an SM to itself (above 128 rows: always)
static int int8_swap(const void* xq, int ldx, const void* wq, int ldw, Int8Out o, Int8Work work, int K, int nb, int parts, bool wide, int mode, int num_sms, cudaStream_t stream) {
  Int8Swap p{};
  p.o = o; p.work = work; p.K = K; p.nb = nb; p.ksplit = parts;
  auto launch = [&](auto kind) {
    constexpr int KIND = decltype(kind)::value;
    if (mode == I8_PLAIN) return swap_launch<I8_PLAIN, KIND>(xq, wq, p, ldx, ldw, wide, num_sms, stream);
    if (mode == I8_RESIDUAL) return swap_launch<I8_RESIDUAL, KIND>(xq, wq, p, ldx, ldw, wide, num_sms, stream);
    if (mode == I8_RELU2) return swap_launch<I8_RELU2, KIND>(xq, wq, p, ldx, ldw, wide, num_sms, stream);
    return swap_launch<I8_GATED, KIND>(xq, wq, p, ldx, ldw, wide, num_sms, stream);
  };
  if (o.kind == DT_F32) return launch(std::integral_constant<int, DT_F32>{});
  return o.kind == DT_BF16 ? launch(std::integral_constant<int, DT_BF16>{}) : launch(std::integral_constant<int, DT_F16>{});
}

static int up16(int k) { return (k + 15) / 16 * 16; }

// result, residual and scales; rows of four features in one access where the row pitch and both addresses allow it
static Int8Out out_of(void* out, const void* residual, const float* xs, const float* ws, int kind, int N, int mode) {
  Int8Out o{out, residual, xs, ws, kind, N, mode == I8_GATED ? N / 2 : N, 0};
  const uintptr_t step = (kind == DT_F32 ? 4 : 2) * (mode == I8_GATED ? 2 : 4);
  o.wide = N % 4 == 0 && (((uintptr_t)out | (uintptr_t)residual) & (step - 1)) == 0;
  return o;
}

}  // namespace jl

using namespace jl;

// the activations' values (rows on 16 bytes) and scales
static size_t values_bytes(int rows, int K) { return rows < 0 || K < 1 ? 0 : ((size_t)rows * up16(K) + 255) / 256 * 256 + (size_t)rows * 4; }
extern "C" JL_API size_t jl_linear_int8_scratch_bytes(int M, int N, int K) { return int8_vec_takes(M, N, K) ? 0 : values_bytes(M, K); }

extern "C" JL_API size_t jl_experts_int8_scratch_bytes(int T, int N, int K) { return int8_vec_takes_pairs(T, N, K) ? 0 : values_bytes(T, K); }

extern "C" JL_API int jl_linear_int8(const void* x, int dtype, int M, int K, long long ldx, const void* wq, int ldw, const float* ws, int N, const void* gain, float eps,
                                     const void* residual, void* out, int out_dtype, int mode, void* scratch, size_t scratch_bytes, int resident, int num_sms, void* stream) {
  JL_CHECK_ARG(dtype >= DT_BF16 && dtype <= DT_F16 && out_dtype >= DT_BF16 && out_dtype <= DT_F16, "jl_linear_int8: element types %d, %d", dtype, out_dtype);
  JL_CHECK_ARG(M >= 0 && M <= I8_MAX_ROWS && N >= 1 && N <= I8_MAX_ROWS && K >= 1 && K <= I8_MAX_K && (ldx >= K || M <= 1), "jl_linear_int8: M=%d N=%d K=%d (at most %d), pitch %lld",
               M, N, K, I8_MAX_K, ldx);
  JL_CHECK_ARG(ldw >= K && ldw % 16 == 0 && ((uintptr_t)wq & 15) == 0, "jl_linear_int8: weights on 16-byte rows (pitch %d)", ldw);
  JL_CHECK_ARG(mode >= I8_PLAIN && mode <= I8_RELU2 && (mode == I8_RESIDUAL) == (residual != nullptr) && (mode != I8_GATED || N % 2 == 0),
               "jl_linear_int8: mode %d with%s residual, N=%d", mode, residual != nullptr ? "" : "out", N);
  if (M == 0) return JL_OK;
  if (num_sms <= 0) num_sms = SMS;
  if (int8_vec_takes(M, N, K)) {
    const Int8Out o = out_of(out, residual, nullptr, ws, out_dtype, N, mode);
    return int8_vec(x, dtype, M > 1 ? ldx : K, gain, eps, wq, ldw, o, M, K, mode, resident != 0, num_sms, (cudaStream_t)stream);
  }
  JL_CHECK_ARG(scratch != nullptr && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= jl_linear_int8_scratch_bytes(M, N, K), "jl_linear_int8: scratch of %zu bytes", scratch_bytes);
  const int ldq = up16(K);
  float* xs = reinterpret_cast<float*>((uint8_t*)scratch + ((size_t)M * ldq + 255) / 256 * 256);
  int rc;
  if ((rc = int8_rows(x, dtype, M, K, ldx, nullptr, M, gain, eps, scratch, ldq, xs, resident ? 2 : 1, (cudaStream_t)stream))) return rc;
  const Int8Out o = out_of(out, residual, xs, ws, out_dtype, N, mode);
  const Int8Work work{nullptr, 1, M, 0, 0};
  const Int8Cut cut = i8s_cut(M, N, K, num_sms);
  if (cut.pieces > 0) {
    const int nb = ((M + cut.pieces - 1) / cut.pieces + 15) / 16 * 16;
    return int8_swap(scratch, ldq, wq, ldw, o, work, K, nb, cut.parts, cut.wide != 0, mode, num_sms, (cudaStream_t)stream);
  }
  return int8_pair(scratch, ldq, wq, ldw, o, work, K, mode, num_sms, (cudaStream_t)stream);
}

extern "C" JL_API int jl_experts_int8(const void* x, int dtype, int M, int K, long long ldx, const int* rows, int T, const int* offsets, int experts, const void* wq, int ldw,
                                      const float* ws, int N, void* out, int out_dtype, int mode, void* scratch, size_t scratch_bytes, int num_sms, void* stream) {
  JL_CHECK_ARG(dtype >= DT_BF16 && dtype <= DT_F16 && out_dtype >= DT_BF16 && out_dtype <= DT_F16, "jl_experts_int8: element types %d, %d", dtype, out_dtype);
  JL_CHECK_ARG(M >= 0 && T >= 0 && T <= I8_MAX_ROWS && N >= 1 && K >= 1 && K <= I8_MAX_K && (ldx >= K || M <= 1) && (rows != nullptr || T <= M),
               "jl_experts_int8: M=%d T=%d N=%d K=%d (at most %d), pitch %lld", M, T, N, K, I8_MAX_K, ldx);
  JL_CHECK_ARG(experts >= 1 && experts <= I8_MAX_EXPERTS && offsets != nullptr, "jl_experts_int8: %d experts (at most %d)", experts, I8_MAX_EXPERTS);
  JL_CHECK_ARG((long long)N * experts < (1ll << 31), "jl_experts_int8: %d x %d weight rows", experts, N);
  JL_CHECK_ARG(ldw >= K && ldw % 16 == 0 && ((uintptr_t)wq & 15) == 0, "jl_experts_int8: weights on 16-byte rows (pitch %d)", ldw);
  JL_CHECK_ARG(mode == I8_PLAIN || mode == I8_RELU2 || (mode == I8_GATED && N % 2 == 0), "jl_experts_int8: mode %d, N=%d", mode, N);
  if (T == 0) return JL_OK;
  if (num_sms <= 0) num_sms = SMS;
  if (int8_vec_takes_pairs(T, N, K)) {
    const Int8Out o = out_of(out, nullptr, nullptr, ws, out_dtype, N, mode);
    return int8_vec_pairs(x, dtype, M, M > 1 ? ldx : K, rows, T, offsets, nullptr, 1, experts, wq, ldw, o, K, mode, num_sms, (cudaStream_t)stream);
  }
  JL_CHECK_ARG(scratch != nullptr && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= values_bytes(T, K),
               "jl_experts_int8: scratch of %zu bytes", scratch_bytes);
  const int ldq = up16(K);
  float* xs = reinterpret_cast<float*>((uint8_t*)scratch + ((size_t)T * ldq + 255) / 256 * 256);
  int rc;
  if ((rc = int8_rows(x, dtype, M, K, ldx, rows, T, nullptr, 0.0f, scratch, ldq, xs, 1, (cudaStream_t)stream))) return rc;
  const Int8Out o = out_of(out, nullptr, xs, ws, out_dtype, N, mode);
  const Int8Work work{offsets, experts, T, 0, 0};
  // Rows of a tile by the rows that an expert has if all have the same (us with 16, 32, 64, 128 rows | pairs, 32 experts of 2048 x 2048: 2 rows 18.6, 17.9, 16.9, 16.9 | 25.8; 32
  // rows 29.6, 25.9, 26.7, 28.0 | 40.6; 64 rows 43.6, 32.1, 29.1, 33.5 | 38.4; 128 rows 77.6, 48.1, 38.2, 41.8 | 42.9; 256 rows 145, 83, 60.4, 63.5 | 56.9); 16 wherever that
  // gives no more tiles than there are slots (8 experts of 1024 x 512, 50 rows: 7.2, 7.5, 9.2, 12.7 | 13.8).
  const int even = (T + experts - 1) / experts;
  const long long tiles = (N + I8S_BM - 1) / I8S_BM * i8_pieces(work, 16);
  if (even > 160 && tiles > 2 * num_sms) return int8_pair(scratch, ldq, wq, ldw, o, work, K, mode, num_sms, (cudaStream_t)stream);
  const int nb = tiles <= 2 * num_sms || even <= 1 ? 16 : even <= 24 ? 32 : 64;
  const int parts = i8s_parts((N + I8S_BM - 1) / I8S_BM * i8_pieces(work, nb), (K + I8S_BK - 1) / I8S_BK, I8S_PARTS, i8s_slots(num_sms));
  return int8_swap(scratch, ldq, wq, ldw, o, work, K, nb, parts, false, mode, num_sms, (cudaStream_t)stream);
}

extern "C" JL_API int jl_choice_int8(const void* x, int dtype, int M, int K, long long ldx, const int* choice, int top, int experts, const void* wq, int ldw, const float* ws, int N,
                                     void* out, int out_dtype, int mode, int num_sms, void* stream) {
  JL_CHECK_ARG(dtype >= DT_BF16 && dtype <= DT_F16 && out_dtype >= DT_BF16 && out_dtype <= DT_F16, "jl_choice_int8: element types %d, %d", dtype, out_dtype);
  JL_CHECK_ARG(M >= 0 && top >= 1 && (long long)M * top <= I8_MAX_ROWS && N >= 1 && K >= 1 && int8_vec_holds_pairs(M * top, K) && (ldx >= K || M <= 1),
               "jl_choice_int8: M=%d top=%d N=%d K=%d, pitch %lld (at most 8 rows of 16384)", M, top, N, K, ldx);
  JL_CHECK_ARG(experts >= 1 && experts <= I8_MAX_EXPERTS && (long long)N * experts < (1ll << 31) && choice != nullptr, "jl_choice_int8: %d experts (at most %d), %d features", experts,
               I8_MAX_EXPERTS, N);
  JL_CHECK_ARG(ldw >= K && ldw % 16 == 0 && ((uintptr_t)wq & 15) == 0, "jl_choice_int8: weights on 16-byte rows (pitch %d)", ldw);
  JL_CHECK_ARG(mode == I8_PLAIN || mode == I8_RELU2 || (mode == I8_GATED && N % 2 == 0), "jl_choice_int8: mode %d, N=%d", mode, N);
  if (M == 0) return JL_OK;
  const Int8Out o = out_of(out, nullptr, nullptr, ws, out_dtype, N, mode);
  return int8_vec_pairs(x, dtype, M, M > 1 ? ldx : K, nullptr, M * top, nullptr, choice, top, experts, wq, ldw, o, K, mode, num_sms > 0 ? num_sms : SMS, (cudaStream_t)stream);
}
