// Products of 8-bit integers for up to eight rows of activations: bound by the weights' way from memory, once.
//
// A unit is 16 features; the eight warps of a CTA take 256-column pieces of K in turn, straight from memory into the registers of `mma.sync.m16n8k32.s8` (weights are its
// 16 rows, activations its 8 columns).  The order of K within an instruction is free as long as both operands have the same: a thread takes 16 neighbouring bytes of a row
// where the instruction's table names 4 + 4 + 4 + 4 apart, so all accesses are 16 bytes.  Two pieces, 8 KB a warp, are under way while one is multiplied, across
// units; the warps' partial sums meet in shared memory, one barrier a unit, whole numbers, in any order the same.
// Every CTA brings the activations to 8 bits itself while its first weights are under way, which saves a launch.
// Bound by latency, then the weights: one B200, us in a chain of cold weights, 1 x 64 x 256 2.5, 1 x 64 x 4096 3.0, 1 x 2048 x 4096 gated 3.9, 1 x 4096 x 4096 5.3 (2.6 at the memory's rate); behind a
// norm a pass over the row more, 1 x 64 x 4096 4.4, 1 x 6144 x 4096 8.5 (3.8), 8 x 2048 x 2048 9.95 (5.4 without).
// A mixture of experts: a CTA has one of up to eight rows and finds whose it is; a token's four of 32 experts of 2048 x 2048 7.7, by choice 7.2 (2.6 at the memory's rate): its weights wait for the router.
// One CTA an SM, which would let the next launch's first weights in, streams too little: 1 x 28672 x 4096 22 -> 35.
#include "int8.cuh"
#include "jllama_b200.h"

namespace jl {

constexpr int I8V_THREADS = 256, I8V_WARPS = 8, I8V_ROWS = 8, I8V_FEATURES = 16, I8V_PIECE = 256;
constexpr int I8V_FUSED = 16384;
constexpr int I8V_SMEM = 96 * 1024;      // (values and fp32 rows of that many elements: 84 KB)

struct Int8Vec {
  Int8Out o;
  const int8_t* wq;
  const void* x;                    // activations, row pitch ldx, normed by gain if given
  const void* gain;
  long long ldx;
  int rows, K, ldw, units, pieces;  // units of features; pieces of a warp
  float eps;
  int early;                        // weights may be read ahead of the wait for the kernels before
  // the form for few rows of a mixture of experts: a CTA has one of `pairs` rows (blockIdx.y) and its expert's weights; `rows` is 1
  const int* offsets;               // [experts + 1], as Int8Work
  const int* index;                 // [pairs] rows of x, or nullptr: the pair's own
  const int* choice;                // [pairs] experts, in any order, instead of offsets and index: the row of x is pair / top
  int experts, pairs, there, top;   // there: rows of x
};

__device__ __forceinline__ void i8v_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__host__ __device__ constexpr int i8v_pitch(int K) { return (K + 127) / 128 * 128 + 64; }      // rows in shared memory: two rows of 64 bytes meet all banks

template <typename T, int MODE, bool EXPERTS>
__global__ void __launch_bounds__(I8V_THREADS, 2) int8_vec_kernel(const Int8Vec p) {
  extern __shared__ __align__(16) uint8_t i8v_smem[];
  __shared__ int parts[2][I8V_WARPS][I8V_ROWS][I8V_FEATURES];
  __shared__ float row_scale[I8V_ROWS];
  __shared__ uint32_t red[I8V_WARPS];
  __shared__ float red_f[I8V_THREADS];
  int8_t* const xs = reinterpret_cast<int8_t*>(i8v_smem);                                 // [rows][pitch]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int pitch = i8v_pitch(p.K), units = p.units;
  pdl_launch_dependents();

  Int8Out out = p.o;
  const int8_t* weights = p.wq;
  const T* source = reinterpret_cast<const T*>(p.x);
  int first = 0;                                                 // row of the result
  bool real = true, nobody = false;                              // the row is there (an index that x does not have is a row of zeros); no expert's: zeros
  if constexpr (EXPERTS) {
    first = blockIdx.y;
    int e, row;
    if (p.choice != nullptr) {
      pdl_wait();
      e = __ldcg(p.choice + first);
      row = first / p.top;
      nobody = (unsigned)e >= (unsigned)p.experts;
      if (nobody) { e = 0; row = -1; }
    } else {
      __shared__ int holder;
      if (threadIdx.x == 0) holder = -1;
      __syncthreads();
      pdl_wait();
      row = p.index != nullptr ? __ldcg(p.index + first) : first;
      const Int8Work work{p.offsets, p.experts, p.pairs, 0, 0};
      for (int i = threadIdx.x; i < p.experts; i += I8V_THREADS)
        if (i8_offset(work, i) <= first && first < i8_offset(work, i + 1)) holder = i;      // (one, where offsets rise)
      __syncthreads();
      e = holder;
      if (e < 0) return;                                         // a row of no expert is left as it was
    }
    weights += (size_t)e * p.o.N * p.ldw;
    out.ws += (size_t)e * p.o.N;
    real = (unsigned)row < (unsigned)p.there;
    if (real) source += (long long)row * p.ldx;
  }

  // ---- the stream of this warp's pieces: unit after unit
  int u_load = blockIdx.x, j_load = 0;
  const int8_t *w_lo, *w_hi;                                     // rows g and g + 8 of the unit
  auto place = [&]() {
    const int f = u_load * I8V_FEATURES + g, last = p.o.N - 1;
    w_lo = weights + (size_t)min(f, last) * p.ldw + 16 * t4;
    w_hi = weights + (size_t)min(f + 8, last) * p.ldw + 16 * t4;
  };
  auto load = [&](uint4 (&buf)[8]) {
    const int c0 = (j_load * I8V_WARPS + warp) * I8V_PIECE;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int c = c0 + 64 * b;
      const bool in = u_load < units && c + 16 * t4 < p.K;
      buf[b] = in ? ldg_stream(w_lo + c) : make_uint4(0, 0, 0, 0);
      buf[4 + b] = in ? ldg_stream(w_hi + c) : make_uint4(0, 0, 0, 0);
    }
    if (++j_load == p.pieces) { j_load = 0; u_load += gridDim.x; place(); }
  };
  place();
  uint4 buf0[8], buf1[8];
  if (!EXPERTS && !p.early) pdl_wait();
  load(buf0);
  load(buf1);
  if (!EXPERTS && p.early) pdl_wait();

  // ---- the activations' rows in 8 bits: 8 / R' warps a row, R' = 1, 2, 4, 8
  {
    const int R = EXPERTS ? 1 : p.rows, per = R <= 1 ? 8 : R <= 2 ? 4 : R <= 4 ? 2 : 1;            // warps of a row
    const int row = warp / per, n = per * 32, i0 = threadIdx.x - row * n;
    const bool there = row < R;
    const T* x = source + (there ? (long long)row * p.ldx : 0);
    const T* gain = reinterpret_cast<const T*>(p.gain);
    constexpr int VE = 16 / sizeof(T);
    // once from memory, all loads at once; what a thread keeps of the row it alone reads again
    T* const raw = reinterpret_cast<T*>(i8v_smem + (size_t)R * pitch) + (size_t)row * ((p.K + VE - 1) / VE * VE);
    const bool whole = p.K % VE == 0 && (p.ldx * (long long)sizeof(T)) % 16 == 0 && (((uintptr_t)p.x | (uintptr_t)p.gain) & 15) == 0;
    uint32_t m = 0;
    float norm = 1.0f;
    if (there && whole) {
      for (int i = i0 * VE; i < p.K; i += 4 * n * VE) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = real && i + u * n * VE < p.K ? *reinterpret_cast<const uint4*>(x + i + u * n * VE) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (i + u * n * VE >= p.K) break;
          *reinterpret_cast<uint4*>(raw + i + u * n * VE) = v[u];
          float f[VE];
          i8r_unpack<T>(v[u], f);
#pragma unroll
          for (int e = 0; e < VE; ++e) m = max(m, i8r_bits(f[e]));
        }
      }
    } else if (there) {
      // element by element; a thread's places are those of its pieces
      for (int i = i0 * VE; i < p.K; i += n * VE)
        for (int e = 0; e < VE && i + e < p.K; ++e) { raw[i + e] = real ? x[i + e] : T(0.0f); m = max(m, i8r_bits(to_f(raw[i + e]))); }
    }
    // the piece at i; columns behind K are zeros
    auto held = [&](int i, float (&f)[VE]) {
      if (whole) {
        i8r_unpack<T>(*reinterpret_cast<const uint4*>(raw + i), f);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = i + e < p.K ? to_f(raw[i + e]) : 0.0f;
      }
    };
    if (!EXPERTS && gain != nullptr) {
      // the sum of squares in the order of i8r_join: a thread has at most 16 pieces (I8V_FUSED), four times four; the first and third four meet, the second and fourth
      float first[4] = {}, second[4] = {};
      bool odd = false;
      for (int i = i0 * VE; there && i < p.K; i += 4 * n * VE, odd = !odd) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (i + u * n * VE >= p.K) break;
          float f[VE];
          held(i + u * n * VE, f);
          const float s = i8r_squares(f);
          first[u] = __fadd_rn(first[u], odd ? 0.0f : s);
          second[u] = __fadd_rn(second[u], odd ? s : 0.0f);
        }
      }
      red_f[threadIdx.x] = __fadd_rn(__fadd_rn(__fadd_rn(first[0], second[0]), __fadd_rn(first[2], second[2])), __fadd_rn(__fadd_rn(first[1], second[1]), __fadd_rn(first[3], second[3])));
      __syncthreads();
      const float* mine = red_f + row * n + lane;
      const float sum = warp_sum(i8r_join<0, 1, I8V_WARPS>([&](auto w) { return decltype(w)::value < per ? mine[32 * decltype(w)::value] : 0.0f; }));
      norm = 1.0f / sqrtf(sum / (float)p.K + p.eps);
    }
    // .. normed
    auto piece = [&](int i, float (&f)[VE]) {
      held(i, f);
      if (EXPERTS || gain == nullptr) return;
      float w[VE];
      if (whole) {
        i8r_unpack<T>(*reinterpret_cast<const uint4*>(gain + i), w);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) w[e] = i + e < p.K ? to_f(gain[i + e]) : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = f[e] * norm * w[e];
    };
    if (!EXPERTS && gain != nullptr) {
      m = 0;
      if (there) {
        for (int i = i0 * VE; i < p.K; i += n * VE) {
          float f[VE];
          piece(i, f);
#pragma unroll
          for (int e = 0; e < VE; ++e) m = max(m, i8r_bits(f[e]));
        }
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = 0;
    for (int i = 0; i < per; ++i) m = max(m, red[row * per + i]);
    // (maxima were taken on fp32 bits)
    const Int8Quotient quotient(__uint_as_float(m));
    const float amax = quotient.amax;
    const Int8Pairs pairs(amax);
    const bool ordinary = quotient.ordinary();
    if (there) {
      int8_t* q = xs + (size_t)row * pitch;
      for (int i = i0 * VE; i < p.K; i += n * VE) {
        float f[VE];
        piece(i, f);
        uint32_t b[VE];
        if (!ordinary) {
#pragma unroll 1
          for (int e = 0; e < VE; ++e) q[i + e] = (int8_t)(quotient(f[e]) & 0xffu);
          continue;
        }
        if (EXPERTS || gain == nullptr) i8r_piece<T, true>(pairs, amax, f, b);
        else i8r_piece<T, false>(pairs, amax, f, b);
        if constexpr (VE == 8) *reinterpret_cast<uint2*>(q + i) = make_uint2(i8r_pack4(b[0], b[1], b[2], b[3]), i8r_pack4(b[4], b[5], b[6], b[7]));
        else *reinterpret_cast<uint32_t*>(q + i) = i8r_pack4(b[0], b[1], b[2], b[3]);
      }
      for (int i = (p.K + VE - 1) / VE * VE + i0; i < pitch; i += n) q[i] = 0;
      if (i0 == 0) row_scale[row] = quotient.scale();
    }
    __syncthreads();
  }

  // ---- products
  int it = 0;
  const bool mine = g < p.rows;
  const int8_t* xrow = xs + (size_t)g * pitch + 16 * t4;
  for (int u = blockIdx.x; u < units; u += gridDim.x, ++it) {
    int acc[2][4] = {};
    auto step = [&](uint4 (&buf)[8], int j) {
      const int c0 = (j * I8V_WARPS + warp) * I8V_PIECE;
      uint4 b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 64 * i;
        b[i] = mine && c + 16 * t4 < p.K ? *reinterpret_cast<const uint4*>(xrow + c) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        i8v_mma(acc[0], buf[i].x, buf[4 + i].x, buf[i].y, buf[4 + i].y, b[i].x, b[i].y);
        i8v_mma(acc[1], buf[i].z, buf[4 + i].z, buf[i].w, buf[4 + i].w, b[i].z, b[i].w);
      }
      load(buf);
    };
    // the two buffers take turns over all pieces of all units
    int j = 0;
    if ((it * p.pieces) & 1) { step(buf1, j); ++j; }
    for (; j + 1 < p.pieces; j += 2) { step(buf0, j); step(buf1, j + 1); }
    if (j < p.pieces) step(buf0, j);
    int(&part)[I8V_WARPS][I8V_ROWS][I8V_FEATURES] = parts[it & 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][2 * t4 + (i & 1)][g + 8 * (i >> 1)] = acc[0][i] + acc[1][i];
    __syncthreads();
    if (threadIdx.x < 32) {                                       // four features of a row a thread
      const int r = threadIdx.x >> 2, f = (threadIdx.x & 3) * 4, f0 = u * I8V_FEATURES + f;
      if (r < p.rows && f0 < p.o.N) {
        int sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < I8V_WARPS; ++w) {
          const int4 v = *reinterpret_cast<const int4*>(&part[w][r][f]);
          sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
        }
        float sw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sw[i] = f0 + i < p.o.N && !nobody ? out.ws[f0 + i] : 0.0f;
        Int8Four<-1> r4;
        if constexpr (MODE == I8_RESIDUAL) r4.load(out, first + r, f0);
        i8_finish4<MODE>(out, first + r, f0, sum, row_scale[r], sw, r4);
      }
    }
  }
}

template <typename T, int MODE, bool EXPERTS = false>
static int vec_launch(const Int8Vec& p, size_t smem, int num_sms, cudaStream_t stream) {
  auto kern = int8_vec_kernel<T, MODE, EXPERTS>;
  // equal shares: as many CTAs as give each the same number of units, up to two an SM
  const int slots = 2 * num_sms / (EXPERTS ? p.pairs : 1), rounds = (p.units + slots - 1) / slots, grid = (p.units + rounds - 1) / rounds;
  JL_CUDA((i8_room<int8_vec_kernel<T, MODE, EXPERTS>, I8V_SMEM>()));
  JL_CUDA(launch_pdl(kern, dim3((unsigned)grid, EXPERTS ? p.pairs : 1), dim3(I8V_THREADS), smem, stream, p));
  return JL_OK;
}

// Whether a product of `rows` rows runs here: what the CTAs bring to 8 bits is little, and the weights are (with many, the tcgen05 kernel's deeper queue earns its second launch:
// us here | there, the rows' kernel included: 1 x 4096 x 4096 6.2 | 7.2, 1 x 6144 x 4096 8.0 | 8.4, 8 x 2048 x 2048 6.7 | 8.0; 1 x 28672 x 4096 21.2 | 20.1, 4 x 4096 x 4096
// 8.6 | 7.7, 8 x 8192 x 2048 9.1 | 7.7).  The host issues one launch here, two there.
bool int8_vec_takes(int rows, int N, int K) {
  return rows <= I8V_ROWS && (rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8) * (long long)K <= I8V_FUSED && (long long)N * K <= (rows <= 2 ? 1 << 25 : 1 << 23);
}

static Int8Vec vec_of(const void* x, long long ldx, const void* gain, float eps, const void* wq, int ldw, const Int8Out& o, int rows, int K, bool early) {
  Int8Vec p{};
  p.o = o;
  p.wq = (const int8_t*)wq; p.x = x; p.gain = gain; p.ldx = ldx; p.rows = rows; p.K = K; p.ldw = ldw; p.eps = eps; p.early = early;
  p.units = (o.N + I8V_FEATURES - 1) / I8V_FEATURES;
  p.pieces = (K + I8V_PIECE * I8V_WARPS - 1) / (I8V_PIECE * I8V_WARPS);
  return p;
}
// values, and the rows themselves
static size_t vec_smem(int rows, int K, int dtype) { return (size_t)rows * (i8v_pitch(K) + (K + 7) / 8 * 8 * (dtype == DT_F32 ? 4 : 2)); }

int int8_vec(const void* x, int dtype, long long ldx, const void* gain, float eps, const void* wq, int ldw, Int8Out o, int rows, int K, int mode, bool early, int num_sms,
             cudaStream_t stream) {
  const Int8Vec p = vec_of(x, ldx, gain, eps, wq, ldw, o, rows, K, early);
  const size_t smem = vec_smem(rows, K, dtype);
  JL_DISPATCH_INT8(dtype, {
    if (mode == I8_PLAIN) return vec_launch<T, I8_PLAIN>(p, smem, num_sms, stream);
    if (mode == I8_RESIDUAL) return vec_launch<T, I8_RESIDUAL>(p, smem, num_sms, stream);
    if (mode == I8_RELU2) return vec_launch<T, I8_RELU2>(p, smem, num_sms, stream);
    return vec_launch<T, I8_GATED>(p, smem, num_sms, stream);
  });
}

// Whether `pairs` rows of a mixture of experts can run here
bool int8_vec_holds_pairs(int pairs, int K) { return pairs <= I8V_ROWS && K <= I8V_FUSED; }

// Whether they do (us here | there, gated: of 32 experts of 2048 x 2048 1 pair 5.7 | 7.7, 4 8.6 | 10.0, 8 11.1 | 12.3, 16 15.6 | 13.7; of 128 of 1536 x
// 2048 8 10.1 | 11.7; of 8 of 8192 x 4096 2 16.0 | 17.2, 4 23.2 | 21.7; 4096 x 14336 1 16.7 | 16.6).
bool int8_vec_takes_pairs(int pairs, int N, int K) { return int8_vec_holds_pairs(pairs, K) && (long long)pairs * N * K <= 1 << 26; }

// `pairs` rows, row index[i] of x [M, K] (or row i) with the weights of the expert whose offsets hold i; or row i / top with those of expert choice[i]
int int8_vec_pairs(const void* x, int dtype, int M, long long ldx, const int* index, int pairs, const int* offsets, const int* choice, int top, int experts, const void* wq, int ldw, Int8Out o, int K, int mode,
                   int num_sms, cudaStream_t stream) {
  Int8Vec p = vec_of(x, ldx, nullptr, 0.0f, wq, ldw, o, 1, K, false);
  p.offsets = offsets; p.index = index; p.choice = choice; p.top = top; p.experts = experts; p.pairs = pairs; p.there = M;
  const size_t smem = vec_smem(1, K, dtype);
  JL_DISPATCH_INT8(dtype, {
    if (mode == I8_PLAIN) return vec_launch<T, I8_PLAIN, true>(p, smem, num_sms, stream);
    if (mode == I8_RELU2) return vec_launch<T, I8_RELU2, true>(p, smem, num_sms, stream);
    return vec_launch<T, I8_GATED, true>(p, smem, num_sms, stream);
  });
}

}  // namespace jl
