// Products of 8-bit integers over many rows on CTA pairs: tiles of 256 rows x 256 features by `tcgen05.mma.cta_group::2.kind::i8` (256 x 256 x 32 an instruction).
//
// Two CTAs of a cluster are one MMA engine: each stages its 128 rows of activations and its 128 rows of weights (32 KB a k-block of 128 bytes), the leader's one thread
// issues for both, each keeps the int32 sums of its own 128 rows in its own TMEM, two accumulators of 256 columns.  A lane of the epilogue holds a row, a column a feature:
// the row's scale is a register, the features' scales come from shared memory (a warp of its own brings both ahead of the tile); finished rows of 128 bytes go through shared
// memory, so that a warp's stores are whole lines.
// Bound by the products and, in seconds of them, the power cap: one B200, us, 2048 x 9216 x 4096 60 (54 without loads, 47 without products), 8192 x 28672 x 4096 gated 718 (2680 TOP/s at
// 1.45 GHz); with few k-blocks by the epilogue: 8192 x 2048 x 128 13.9 (18.5 with scales from memory in the epilogue), gated 8192 x 4096 x 128 27 (32; 36 with a true quotient per
// gate; issue slots 43 %, tensor pipe 6 %: eight warps, each one chain from
// accumulator to store).  Rings of 3, 4, 5 stages: 2048 x 9216 x 4096 69, 62, 59; six gave nothing more.
// One matrix, or one per expert (rows ordered by expert, at any row): what a tile holds of the next expert's rows is computed and not stored.  (Rows of
// several experts held once and gathered by the loads, `tile::gather4`: 8192 tokens x 4 of 32 experts of 2048 x 2048 410 us, with the rows written out by the kernel that
// brings them to 8 bits 144.)
#include <atomic>

#include "int8.cuh"
#include "jllama_b200.h"
#include "tcgen05.cuh"

namespace jl {

constexpr int I8P_BM = 128, I8P_BN = 256, I8P_BK = 128, I8P_THREADS = 384;      // rows per CTA; features per pair; warps: 0 TMA, 1 MMA (leader), 2 TMEM, 3 list and scales, 4-11 results
constexpr uint32_t I8P_A_BYTES = I8P_BM * I8P_BK;
constexpr uint32_t I8P_EPI = 8 * 4096;                     // of each epilogue warp: 32 rows of 128 bytes
constexpr uint32_t I8P_SCALES = (I8P_BN + I8P_BM) * 4;     // of a tile: its features', its rows'
constexpr int I8P_STAGES = 8;                              // at most
constexpr size_t I8P_SMEM = 227 * 1024;
constexpr uint32_t I8P_LEADER = 0xFEFFFFFFu;               // shared::cluster address of the same offset in CTA 0

struct Int8Pair {
  Int8Out o;
  Int8Work work;
  int K, stages, bn;              // bn: features of a tile, a multiple of 32
  uint32_t idesc;
};

__device__ __forceinline__ uint32_t i8p_mapa(uint32_t local_smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local_smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void i8p_remote_arrive(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void i8p_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a load by either CTA; its bytes count on the leader's mbarrier
__device__ __forceinline__ void i8p_load(uint32_t smem_dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, uint64_t hint) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & I8P_LEADER), "r"(c0), "r"(c1), "l"(hint)
      : "memory");
}
__device__ __forceinline__ void i8p_mma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void i8p_commit_both(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t i8p_pack(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16(a, b);
  }
}

// `rows` rows of up to 128 bytes, `cols` elements of them, between a warp's buffer (chunks of 16 bytes turned by the row) and rows of memory on any boundary: neighbouring lanes
// have neighbouring words.  (2924 x 11962 x 112 + residual 71 us; a row a lane, element by element, 152.)
template <typename Word, bool OUT, typename T>
__device__ __forceinline__ void i8p_words(uint8_t* buffer, T* memory, int pitch, int rows, int cols, int lane) {
  constexpr int FLY = OUT ? 8 : 32;                                                   // rows under way at once
  constexpr int EACH = sizeof(Word) >= sizeof(T) ? sizeof(Word) / sizeof(T) : 1;      // elements of a word (fp32 has words of four bytes only)
#pragma unroll
  for (int c = 0; c < 128 / (int)sizeof(Word); c += 32) {
    const int byte = (c + lane) * (int)sizeof(Word), col = (c + lane) * EACH;
    if (col >= cols) continue;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += FLY) {
      Word q[FLY];
#pragma unroll
      for (int i = 0; i < FLY; ++i) {
        const int r = r0 + i;
        uint8_t* const at = buffer + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15);
        if constexpr (OUT) q[i] = *reinterpret_cast<const Word*>(at);
        else q[i] = r < rows ? *reinterpret_cast<const Word*>(memory + (size_t)r * pitch + col) : Word(0);
      }
#pragma unroll
      for (int i = 0; i < FLY; ++i) {
        const int r = r0 + i;
        if constexpr (OUT) { if (r < rows) *reinterpret_cast<Word*>(memory + (size_t)r * pitch + col) = q[i]; }
        else *reinterpret_cast<Word*>(buffer + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15)) = q[i];
      }
    }
  }
}

template <typename T, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8P_THREADS, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Int8Pair p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  const int stages = p.stages;
  const uint32_t stage_bytes = I8P_A_BYTES + (uint32_t)p.bn / 2 * I8P_BK, epi_smem = smem_base + stages * stage_bytes;
  const uint32_t scale_smem = epi_smem + I8P_EPI, bars = scale_smem + 2 * I8P_SCALES;        // full[stages] | empty[stages] | tfull[2] | tempty[2] | sfull[2] | sempty[2]
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
  auto tfull_bar = [&](int s) { return bars + 8u * (2 * stages + s); };
  auto tempty_bar = [&](int s) { return bars + 8u * (2 * stages + 2 + s); };
  auto sfull_bar = [&](int s) { return bars + 8u * (2 * stages + 4 + s); };
  auto sempty_bar = [&](int s) { return bars + 8u * (2 * stages + 6 + s); };
  const uint32_t tmem_slot = bars + 8u * (2 * stages + 8);
  uint8_t* const smem = smem_raw + (smem_base - tc::smem_u32(smem_raw));
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - smem_base));
  int* table = reinterpret_cast<int*>(smem + (tmem_slot + 16 - smem_base));
  float* const scales = reinterpret_cast<float*>(smem + (scale_smem - smem_base));      // [2][features' | rows']

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));     // 0 = leader
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int num_kb = (p.K + I8P_BK - 1) / I8P_BK;

  if (warp == 0 && lane == 0) {
    tc::prefetch_tensormap(&tmap_x);
    tc::prefetch_tensormap(&tmap_w);
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(full_bar(s), 2);                        // leader's: its own expect_tx arrive and the other producer's arrive
      tc::mbar_init(empty_bar(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(tfull_bar(s), 1);
      tc::mbar_init(tempty_bar(s), 16);                     // leader's: the eight epilogue warps of both CTAs
      tc::mbar_init(sfull_bar(s), 1);
      tc::mbar_init(sempty_bar(s), 8);
    }
    tc::fence_barrier_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 3) i8_list(p.work, table);
  tc::fence_before_sync();
  i8p_cluster_sync();                                       // barriers of both CTAs are there before the other one uses them
  tc::fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_ptr;
  pdl_wait();
  pdl_launch_dependents();
  const int tiles = table[p.work.experts];

  if (warp == 0) {
    // ===================================================== TMA producer (one per CTA: its halves of both operands)
    if (lane == 0) {
      Int8Walk walk;
      int stage = 0; uint32_t phase = 0;
      for (int t = pair; t < tiles; t += n_pairs) {
        const Int8Tile tile = walk.at(p.work, table, t);
        const int x_row = tile.row0 + (int)rank * I8P_BM, w_row = tile.expert * p.o.N + tile.col * p.bn + (int)rank * (p.bn / 2);
        for (int kb = 0; kb < num_kb; ++kb) {
          tc::mbar_wait(empty_bar(stage), phase ^ 1);
          const uint32_t sa = smem_base + stage * stage_bytes, sb = sa + I8P_A_BYTES;
          if (rank == 0) tc::mbar_expect_tx(full_bar(stage), 2 * stage_bytes);      // both CTAs' bytes
          else i8p_remote_arrive(i8p_mapa(full_bar(stage), 0));
          i8p_load(sa, &tmap_x, full_bar(stage), kb * I8P_BK, x_row, tc::EVICT_NORMAL);
          i8p_load(sb, &tmap_w, full_bar(stage), kb * I8P_BK, w_row, tc::EVICT_LAST);
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ===================================================== MMA issuer: one thread of the leader, for the pair
    if (rank == 0 && lane == 0) {
      int stage = 0, it = 0; uint32_t phase = 0;
      for (int t = pair; t < tiles; t += n_pairs, ++it) {
        const int as = it & 1;
        tc::mbar_wait(tempty_bar(as), ((it >> 1) & 1) ^ 1);      // both CTAs' epilogues have drained this accumulator
        tc::fence_after_sync();
        const uint32_t d = tmem_base + as * I8P_BN;
        for (int kb = 0; kb < num_kb; ++kb) {
          tc::mbar_wait(full_bar(stage), phase);
          tc::fence_after_sync();
          const uint32_t sa = smem_base + stage * stage_bytes;
          const uint64_t da = tc::smem_desc_kmajor_sw128(sa), db = tc::smem_desc_kmajor_sw128(sa + I8P_A_BYTES);
#pragma unroll
          for (int k = 0; k < I8P_BK / 32; ++k) i8p_mma(d, da + 2 * k, db + 2 * k, p.idesc, kb != 0 || k != 0);
          i8p_commit_both(empty_bar(stage));                // frees the slot in both CTAs when these MMAs retire
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
        i8p_commit_both(tfull_bar(as));
      }
    }
  } else if (warp == 3) {
    // ===================================================== scales of a tile, ahead of its epilogue
    Int8Walk walk;
    int it = 0;
    for (int t = pair; t < tiles; t += n_pairs, ++it) {
      const Int8Tile tile = walk.at(p.work, table, t);
      const int as = it & 1, n0 = tile.col * p.bn, first = (int)rank * I8P_BM;
      const float* const ws = p.o.ws + (size_t)tile.expert * p.o.N;
      float fs[I8P_BN / 32], rs[I8P_BM / 32];
#pragma unroll
      for (int i = 0; i < I8P_BN / 32; ++i) fs[i] = n0 + lane + 32 * i < p.o.N ? ws[n0 + lane + 32 * i] : 0.0f;
#pragma unroll
      for (int i = 0; i < I8P_BM / 32; ++i) {
        const int r = first + lane + 32 * i;
        rs[i] = r < tile.rows ? p.o.xs[tile.row0 + r] : 0.0f;
      }
      tc::mbar_wait(sempty_bar(as), ((it >> 1) & 1) ^ 1);
      float* const to = scales + as * (I8P_BN + I8P_BM);
#pragma unroll
      for (int i = 0; i < I8P_BN / 32; ++i) to[lane + 32 * i] = fs[i];
#pragma unroll
      for (int i = 0; i < I8P_BM / 32; ++i) to[I8P_BN + lane + 32 * i] = rs[i];
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(sfull_bar(as));
    }
  } else if (warp >= 4) {
    // ===================================================== results: TMEM -> registers -> shared memory -> whole lines; four warps a half of the features
    const int quarter = warp & 3, part = (warp >> 2) - 1;   // TMEM lanes [32 quarter, 32 quarter + 32)
    uint8_t* const mine = smem + (epi_smem - smem_base) + (warp - 4) * 4096;
    const uint32_t tempty_leader = i8p_mapa(tempty_bar(0), 0);
    constexpr int PER = 128 / sizeof(T);                    // results of a 128-byte row
    constexpr int STEP = MODE == I8_GATED ? 2 * PER : PER;  // accumulator columns for them
    constexpr int AT = MODE == I8_PLAIN && STEP >= 64 ? 2 : 1;      // reads of 32 columns under way at once (two with the rest spill)
    const T* const residual = reinterpret_cast<const T*>(p.o.residual);
    T* const out = reinterpret_cast<T*>(p.o.out);
    // rows off the 16-byte boundary: words of four bytes where two elements fill one in every row
    const bool words = sizeof(T) == 4 || (p.o.ldo % 2 == 0 && (((uintptr_t)out | (uintptr_t)residual) & 3) == 0);
    Int8Walk walk;
    int it = 0;
    for (int t = pair; t < tiles; t += n_pairs, ++it) {
      const Int8Tile tile = walk.at(p.work, table, t);
      const int as = it & 1;
      const int first = (int)rank * I8P_BM + quarter * 32;               // of the tile's rows, this warp's first
      const int n0 = tile.col * p.bn, n_end = min(n0 + p.bn, p.o.N);      // the tile's features
      const int rows = tile.rows - first;                                // how many of its 32 there are
      const size_t row0 = (size_t)tile.row0 + first;
      // residuals: the line of the lane's row, all of it at once, the next one's while this one's results are written
      uint32_t own[MODE == I8_RESIDUAL ? 32 : 1];
      auto bring = [&](int c0) {
        if constexpr (MODE == I8_RESIDUAL) {
          if (!p.o.wide || lane >= rows) return;
          const T* r = residual + (row0 + lane) * p.o.ldo + n0 + c0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint4 q = n0 + c0 + j * (16 / (int)sizeof(T)) < n_end ? reinterpret_cast<const uint4*>(r)[j] : make_uint4(0, 0, 0, 0);
            own[4 * j] = q.x; own[4 * j + 1] = q.y; own[4 * j + 2] = q.z; own[4 * j + 3] = q.w;
          }
        }
      };
      bring(part * STEP);
      tc::mbar_wait(sfull_bar(as), (it >> 1) & 1);
      const float* const ws = scales + as * (I8P_BN + I8P_BM);
      const float sx = ws[I8P_BN + quarter * 32 + lane];
      tc::mbar_wait(tfull_bar(as), (it >> 1) & 1);
      tc::fence_after_sync();
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + as * I8P_BN;
      if (rows > 0) {
#pragma unroll 1
        for (int c0 = part * STEP; n0 + c0 < n_end; c0 += 2 * STEP) {     // the two halves of the warps take turns
          uint32_t w[32];
          if constexpr (MODE == I8_RESIDUAL) {
            if (!p.o.wide) {
              T* const r = const_cast<T*>(residual) + row0 * p.o.ldo + n0 + c0;
              __syncwarp();                                 // what was in the buffer has been read
              if (words) i8p_words<uint32_t, false>(mine, r, p.o.ldo, min(rows, 32), n_end - n0 - c0, lane);
              else i8p_words<uint16_t, false>(mine, r, p.o.ldo, min(rows, 32), n_end - n0 - c0, lane);
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint4 q = *reinterpret_cast<const uint4*>(mine + lane * 128 + ((j ^ (lane & 7)) << 4));
                own[4 * j] = q.x; own[4 * j + 1] = q.y; own[4 * j + 2] = q.z; own[4 * j + 3] = q.w;
              }
            }
          }
#pragma unroll
          for (int h0 = 0; h0 < STEP / 32; h0 += AT) {
            uint32_t v[AT][32];
#pragma unroll
            for (int a = 0; a < AT; ++a) tc::tmem_ld32(t_row + c0 + (h0 + a) * 32, v[a]);
            tc::tmem_ld_wait();
#pragma unroll
            for (int a = 0; a < AT; ++a) {
              const int h = h0 + a, col = n0 + c0 + h * 32;
              float y[32];
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 sw = *reinterpret_cast<const float4*>(ws + c0 + h * 32 + j);
                y[j] = __int2float_rn((int)v[a][j]) * sx * sw.x;
                y[j + 1] = __int2float_rn((int)v[a][j + 1]) * sx * sw.y;
                y[j + 2] = __int2float_rn((int)v[a][j + 2]) * sx * sw.z;
                y[j + 3] = __int2float_rn((int)v[a][j + 3]) * sx * sw.w;
              }
              if constexpr (MODE == I8_RESIDUAL) {       // (__fadd_rn: see i8_finish4)
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  if constexpr (sizeof(T) == 4) {
                    y[j] = __fadd_rn(y[j], __uint_as_float(own[j]));
                  } else {
                    const uint32_t q = own[h * 16 + j / 2];
                    if constexpr (std::is_same_v<T, __half>) y[j] = __fadd_rn(y[j], __half2float(__ushort_as_half((unsigned short)(j & 1 ? q >> 16 : q))));
                    else y[j] = __fadd_rn(y[j], j & 1 ? bf16_hi(q) : bf16_lo(q));
                  }
                }
              }
              if constexpr (MODE == I8_RELU2) {
#pragma unroll
                for (int j = 0; j < 32; ++j) y[j] = i8_relu2(y[j]);
              }
              if constexpr (MODE == I8_GATED) {
#pragma unroll
                for (int j = 0; j < 16; ++j) y[j] = i8_gate(y[2 * j], y[2 * j + 1]);
              }
              constexpr int Y = MODE == I8_GATED ? 16 : 32;     // results of these 32 columns
              if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < Y; ++j) w[h * Y + j] = __float_as_uint(y[j]);
              } else {
#pragma unroll
                for (int j = 0; j < Y / 2; ++j) w[h * Y / 2 + j] = i8p_pack<T>(y[2 * j], y[2 * j + 1]);
              }
            }
          }
          if (n0 + c0 + 2 * STEP < n_end) bring(c0 + 2 * STEP);
          __syncwarp();                                     // what was in the buffer has been read
#pragma unroll
          for (int j = 0; j < 8; ++j)                       // 16-byte chunks, turned by the row so that a warp's accesses meet all banks
            *reinterpret_cast<uint4*>(mine + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
          __syncwarp();
          const int o0 = MODE == I8_GATED ? (n0 + c0) / 2 : n0 + c0, o_end = MODE == I8_GATED ? n_end / 2 : n_end;      // result columns of the 128 bytes
          if (p.o.wide) {
            const int j = lane & 7, col = o0 + j * (16 / (int)sizeof(T));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3);
              const uint4 q = *reinterpret_cast<const uint4*>(mine + r * 128 + ((j ^ (r & 7)) << 4));
              if (r < rows && col < o_end) *reinterpret_cast<uint4*>(out + (row0 + r) * p.o.ldo + col) = q;
            }
          } else {
            T* const o = out + row0 * p.o.ldo + o0;
            if (words) i8p_words<uint32_t, true>(mine, o, p.o.ldo, min(rows, 32), o_end - o0, lane);
            else i8p_words<uint16_t, true>(mine, o, p.o.ldo, min(rows, 32), o_end - o0, lane);
          }
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        i8p_remote_arrive(tempty_leader + 8u * as);         // the leader's
        tc::mbar_arrive(sempty_bar(as));
      }
    }
  }

  tc::fence_before_sync();
  __syncwarp();
  i8p_cluster_sync();                                       // neither CTA frees TMEM or exits while the pair still uses it
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
}

static size_t i8p_smem(int stages, int bn, int experts) { return (size_t)stages * (I8P_A_BYTES + bn / 2 * I8P_BK) + I8P_EPI + 2 * I8P_SCALES + 8 * (2 * stages + 8) + 16 + 4 * i8_table_ints(experts) + 1024; }

using Int8PairKernel = void (*)(const CUtensorMap, const CUtensorMap, const Int8Pair);
template <typename T>
static cudaError_t pair_kernel(int mode, Int8PairKernel* k) {
  if (mode == I8_PLAIN) { *k = int8_pair_kernel<T, I8_PLAIN>; return i8_room<int8_pair_kernel<T, I8_PLAIN>>(); }
  if (mode == I8_RESIDUAL) { *k = int8_pair_kernel<T, I8_RESIDUAL>; return i8_room<int8_pair_kernel<T, I8_RESIDUAL>>(); }
  if (mode == I8_RELU2) { *k = int8_pair_kernel<T, I8_RELU2>; return i8_room<int8_pair_kernel<T, I8_RELU2>>(); }
  *k = int8_pair_kernel<T, I8_GATED>;
  return i8_room<int8_pair_kernel<T, I8_GATED>>();
}

// Clusters that can be resident at once: the tile loop is persistent, a pair that starts when another one is done doubles the time.  Asked once per device.
static int i8p_resident(Int8PairKernel kern, int num_sms) {
  constexpr int DEVICES = 16;
  static std::atomic<int> known[DEVICES];
  int dev = 0, n = 0;
  const bool cached = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < DEVICES;
  if (cached) n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(I8P_THREADS);
    cfg.dynamicSmemBytes = I8P_SMEM;
    cfg.gridDim = dim3((num_sms / 2) * 2);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = num_sms / 2; }
    if (cached) known[dev].store(n, std::memory_order_relaxed);
  }
  return n < num_sms / 2 ? n : num_sms / 2;
}

// Features of a tile: 256, or fewer where that saves more than it costs in rounds of tiles over the pairs.  A k-block takes 406 ns with 256 features, 375 with 192, 345 with
// 128 (2048 x 6144 x 4096): what does not shrink with the features is worth 600 of them.
static int i8p_features(const Int8Out& o, const Int8Work& work, int pairs) {
  const long long pieces = (work.rows + work.chunk - 1) / work.chunk + (work.offsets != nullptr ? work.experts / 2 : 0);
  int best = I8P_BN;
  long long least = 0;
  for (int bn = I8P_BN; bn >= 64; bn -= 32) {
    const long long rounds = (pieces * ((o.N + bn - 1) / bn) + pairs - 1) / pairs, cost = rounds * (bn + 600);
    if (bn == I8P_BN || cost < least) { best = bn; least = cost; }
  }
  return best;
}

int int8_pair(const void* xq, int ldx, const void* wq, int ldw, Int8Out o, Int8Work work, int K, int mode, int num_sms, cudaStream_t stream) {
  Int8Pair p{};
  // 16-byte pieces of rows of results (and residuals)
  const int size = o.kind == DT_F32 ? 4 : 2, out_n = mode == I8_GATED ? o.N / 2 : o.N;
  o.wide = (out_n * size) % 16 == 0 && (((uintptr_t)o.out | (uintptr_t)o.residual) & 15) == 0;
  work.chunk = 2 * I8P_BM;
  Int8PairKernel kern = nullptr;
  JL_DISPATCH_INT8(o.kind, JL_CUDA(pair_kernel<T>(mode, &kern)));
  const int pairs = i8p_resident(kern, num_sms), E = work.experts;
  p.bn = i8p_features(o, work, pairs);
  work.cols = (o.N + p.bn - 1) / p.bn;
  p.o = o; p.work = work; p.K = K;
  p.idesc = tc::idesc_s8_s32(2 * I8P_BM, p.bn);
  const long long most = work.cols * i8_pieces(work, work.chunk);
  JL_CHECK_ARG(most < (1ll << 30), "int8 product: %lld tiles", most);
  CUtensorMap tx, tw;
  int rc;
  if ((rc = make_tmap_2d_i8(&tx, xq, work.rows, K, ldx, I8P_BM))) return rc;
  if ((rc = make_tmap_2d_i8(&tw, wq, (uint64_t)o.N * E, K, ldw, p.bn / 2))) return rc;
  p.stages = I8P_STAGES;
  while (i8p_smem(p.stages, p.bn, E) > I8P_SMEM) --p.stages;
  JL_CUDA(launch_pdl(kern, dim3(2 * (unsigned)(most < pairs ? most : pairs)), dim3(I8P_THREADS), i8p_smem(p.stages, p.bn, E), stream, tx, tw, p));
  return JL_OK;
}

}  // namespace jl
