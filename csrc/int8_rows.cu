// Rows of numbers as int8 values and one scale each: s = amax / 127, q = 127 x / amax rounded to the nearest whole number, ties to even.
//
// Both are what 64 bits would give: s is one rounded quotient, and q is decided exactly (int8.cuh).  A row of zeros has s = 0, a row that holds an infinity or a NaN s = NaN, both
// with q = 0: what such a row is multiplied with gives zeros or NaN.  With gains the row is normed first (RMS, fp32, no rounding in between; the sum of squares in one order, int8.cuh).
//
// One pass over memory: a row's 16-byte pieces stay in registers between its maximum and its values, 2 to 16 a thread; a row has 8 threads, a warp, 128 or 256 threads.  Rows longer than
// registers hold are read twice, an element a thread.  Rows off the 16-byte boundary are taken in pieces of the boundary all the same (the two at the ends element by
// element); a warp then turns its values to the boundary of the result with its neighbours' bytes.
// Bound by memory: one B200, us, 8192 x 14336 bf16 51.7 (6.8 TB/s), 32768 x 2048 29.0 (6.9), 65536 x 512 16.8 (6.0), 2048 x 4096 fp32 7.8 (5.4); with many short rows 65536 x 128 5.6
// (4.5; a warp a row 13.7); off the boundary about twice the time: 4097 x 1001 bf16 5.7, 6753 x 11331 66, 61737 x 45 8.8 (a warp a row 28).  Behind a norm by instructions as well: 1 x 4096 2.1
// (1.4 without), 2048 x 4096 11.4 (7.1), 8192 x 2048 15.3, 8192 x 14336 114 (53); off the boundary 4097 x 1001 14.3, 8192 x 4095 80.
// Maxima are taken on the bits without their sign, as whole numbers: the order is that of the magnitudes, with infinities and NaN above all of them.
#include "int8.cuh"
#include "jllama_b200.h"

namespace jl {

__host__ __device__ constexpr int i8r_threads(int group) { return group < 128 ? 128 : group; }

struct Int8Rows {
  const void* x;
  const int* rows;            // source row of every row of the result, or nullptr: the same
  const void* gain;           // norm first: gains of x's type, or nullptr
  int8_t* q;
  float* s;
  int M, n, K, ldq;           // rows of x, rows of the result, columns, row pitch of q (columns behind K become zeros)
  long long ldx;
  float eps;
  int early;                  // let the next kernel start before this one is done: 1 behind the kernels ahead, 2 at once
};

// G threads' maximum or sum
template <int G>
__device__ __forceinline__ uint32_t i8r_max(uint32_t v, uint32_t* red) {
  if constexpr (G < 32) {
#pragma unroll
    for (int o = G / 2; o > 0; o /= 2) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (G == 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < G / 32; ++i) v = max(v, red[i]);
  return v;
}
// (in the order of i8r_join)
template <int G>
__device__ __forceinline__ float i8r_sum(float v, float* red) {
  if constexpr (G > 32) {
    red[threadIdx.x] = v;
    __syncthreads();
    v = i8r_join<0, 1, G / 32>([&](auto w) { return red[32 * decltype(w)::value + (threadIdx.x & 31)]; });
  }
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A piece that begins `away` elements behind a 16-byte boundary, from the two pieces of the boundary that hold it
template <typename T>
__device__ __forceinline__ uint4 i8r_turn(const uint4& lo, const uint4& hi, int away) {
  uint32_t u[7] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z};
  const int bytes = away * (int)sizeof(T);
  if (bytes & 8) { u[0] = u[2]; u[1] = u[3]; u[2] = u[4]; u[3] = u[5]; u[4] = u[6]; u[5] = hi.w; }
  if (bytes & 4) { u[0] = u[1]; u[1] = u[2]; u[2] = u[3]; u[3] = u[4]; u[4] = u[5]; }
  const int bits = 8 * (bytes & 3);
  return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits), __funnelshift_r(u[2], u[3], bits), __funnelshift_r(u[3], u[4], bits));
}
// The piece from column c on, zeros for what is no column of the row: at once where it ends at or before `whole` (and x + c is on the boundary), element by element at a row's ends
template <typename T>
__device__ __forceinline__ uint4 i8r_load(const T* x, int c, int whole, int K) {
  constexpr int VE = 16 / sizeof(T);
  if (c >= 0 && c + VE <= whole) return *reinterpret_cast<const uint4*>(x + c);
  alignas(16) T e[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) e[i] = c + i >= 0 && c + i < K ? x[c + i] : from_f<T>(0.0f);
  return *reinterpret_cast<const uint4*>(e);
}

// G threads a row, up to NV 16-byte pieces a thread, all on their way at once.
// NV = 0: any row, read again for its values.  EDGE: rows and results on any boundary
template <typename T, int G, int NV, bool NORM, bool EDGE>
__global__ void __launch_bounds__(i8r_threads(G)) int8_rows_kernel(const Int8Rows p) {
  __shared__ uint32_t red_max[i8r_threads(G) / 32];
  __shared__ float red_sum[NORM && G > 32 ? G : 1];
  if (p.early == 2) pdl_launch_dependents();
  pdl_wait();
  if (p.early == 1) pdl_launch_dependents();
  constexpr int VE = 16 / sizeof(T);
  const int t = threadIdx.x % G, lane = threadIdx.x & 31;
  int row = blockIdx.x * (i8r_threads(G) / G) + threadIdx.x / G;
  if (G < 32) row = min(row, p.n - 1);                           // (a warp has several rows and stays whole: the last one may be done twice)
  if (row >= p.n) return;                                        // (whole groups)
  const T* gain = reinterpret_cast<const T*>(p.gain);
  // first element of the row, or nullptr for a row of zeros: one that is not there
  const int src = p.rows != nullptr ? p.rows[row] : row;
  const T* const x = src >= 0 && src < p.M ? reinterpret_cast<const T*>(p.x) + (long long)src * p.ldx : nullptr;
  // behind a norm pieces begin at columns, whatever the boundary (the order of the sum)
  const int away = NORM && (EDGE || NV == 0) ? (int)(((uintptr_t)x & 15) / sizeof(T)) : 0;
  const bool gain_whole = ((uintptr_t)gain & 15) == 0;
  if constexpr (NV > 0) {
    // how many elements the row's first piece has in front of the row, and how many pieces there are
    const int lead = EDGE && !NORM ? (int)(((uintptr_t)x & 15) / sizeof(T)) : 0, pieces = (lead + p.K + VE - 1) / VE;
    uint4 w[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      w[v] = make_uint4(0, 0, 0, 0);
      if (x == nullptr || t + v * G >= pieces + (away > 0)) continue;      // (one more, for the last piece to be turned)
      const int c = (t + v * G) * VE - lead - away;              // its first column
      w[v] = EDGE ? i8r_load(x, c, p.K, p.K) : *reinterpret_cast<const uint4*>(x + c);
    }
    if constexpr (EDGE && NORM) {
      constexpr int W = G < 32 ? G : 32;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        uint4 hi = make_uint4(__shfl_down_sync(0xffffffffu, w[v].x, 1, W), __shfl_down_sync(0xffffffffu, w[v].y, 1, W), __shfl_down_sync(0xffffffffu, w[v].z, 1, W),
                              __shfl_down_sync(0xffffffffu, w[v].w, 1, W));
        if (lane % W == W - 1) hi = away > 0 && t + v * G < pieces ? i8r_load(x, (t + v * G + 1) * VE - away, p.K, p.K) : make_uint4(0, 0, 0, 0);
        w[v] = i8r_turn<T>(w[v], hi, away);
      }
    }
    {
      uint32_t m = 0;
      float norm = 1.0f;
      if constexpr (NORM) {
        const float sum = i8r_join<0, 1, NV>([&](auto v) {
          float f[VE];
          i8r_unpack<T>(w[decltype(v)::value], f);
          return i8r_squares(f);
        });
        norm = 1.0f / sqrtf(i8r_sum<G>(sum, red_sum) / (float)p.K + p.eps);
      }
      auto element = [&](float x0, float g) { return NORM ? x0 * norm * g : x0; };
      auto gains = [&](int v, float (&g)[VE]) {
        if constexpr (NORM) {
          const int c = (t + v * G) * VE;
          if (EDGE ? gain_whole && c + VE <= p.K : t + v * G < pieces) {
            i8r_unpack<T>(*reinterpret_cast<const uint4*>(gain + c), g);
          } else if constexpr (EDGE) {
#pragma unroll
            for (int i = 0; i < VE; ++i) g[i] = c + i < p.K ? to_f(gain[c + i]) : 0.0f;
          }
        }
      };
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if constexpr (NORM) {
          float f[VE], g[VE] = {};
          i8r_unpack<T>(w[v], f);
          gains(v, g);
#pragma unroll
          for (int i = 0; i < VE; ++i) m = max(m, i8r_bits(element(f[i], g[i])));
        } else if constexpr (sizeof(T) == 4) {
          m = max(max(max(m, w[v].x & 0x7fffffffu), w[v].y & 0x7fffffffu), max(w[v].z & 0x7fffffffu, w[v].w & 0x7fffffffu));
        } else {
          m = __vmaxu2(__vmaxu2(__vmaxu2(m, w[v].x & 0x7fff7fffu), w[v].y & 0x7fff7fffu), __vmaxu2(w[v].z & 0x7fff7fffu, w[v].w & 0x7fff7fffu));
        }
      }
      float amax;
      if constexpr (NORM) {
        amax = i8r_value<float>(i8r_max<G>(m, red_max));
      } else {
        if constexpr (sizeof(T) == 2) m = max(m & 0xffffu, m >> 16);
        amax = i8r_value<T>(i8r_max<G>(m, red_max));
      }
      const Int8Quotient quotient(amax);
      int8_t* q = p.q + (size_t)row * p.ldq;
      for (int i = p.K + t; i < p.ldq; i += G) q[i] = 0;
      if (t == 0) p.s[row] = quotient.scale();
      const bool ordinary = quotient.ordinary();
      if (!ordinary) {                                           // zeros, tiny numbers, no numbers: element by element, again from memory
#pragma unroll 1
        for (int i = t; i < p.K; i += G) q[i] = (int8_t)(quotient(x == nullptr ? 0.0f : element(to_f(x[i]), NORM ? to_f(gain[i]) : 0.0f)) & 0xffu);
        if (!(EDGE && G < 32)) return;                           // (a warp's rows turn their values together)
      }
      const Int8Pairs pairs(amax);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (EDGE && G < 32 ? v * G >= (p.K + 2 * VE - 2) / VE : (EDGE ? t - lane : t) + v * G >= pieces) break;        // (EDGE: whole warps)
        float f[VE], g[VE] = {};
        i8r_unpack<T>(w[v], f);
        gains(v, g);
        uint32_t b[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] = element(f[i], g[i]);
        i8r_piece<T, !NORM>(pairs, amax, f, b);
        using Word = std::conditional_t<VE == 8, uint64_t, uint32_t>;
        Word mine = i8r_pack4(b[0], b[1], b[2], b[3]);
        if constexpr (VE == 8) mine |= (Word)i8r_pack4(b[4], b[5], b[6], b[7]) << 32;
        const int c = (t + v * G) * VE - lead;
        if constexpr (!EDGE) {
          *reinterpret_cast<Word*>(q + c) = mine;
        } else {
          // the word of the result that holds this piece's first byte: `turn_by` bytes of the piece before it, then this one's.  Whole words are stored by the lane whose
          // piece begins in them, the bytes of others one by one.
          const int turn_by = (int)((uintptr_t)(q + c) % VE);
          constexpr int W = G < 32 ? G : 32;
          const Word before = __shfl_up_sync(0xffffffffu, mine, 1, W);
          const bool there = t + v * G < pieces && (G >= 32 || ordinary);
          const bool full = there && (lane % W > 0 || turn_by == 0) && c - turn_by >= 0 && c - turn_by + VE <= p.K;
          const bool next = __shfl_down_sync(0xffffffffu, full, 1, W) && lane % W < W - 1;
          if (full) *reinterpret_cast<Word*>(q + c - turn_by) = turn_by == 0 ? mine : (Word)(mine << (8 * turn_by)) | (Word)(before >> (8 * (VE - turn_by)));
          if (there && (!full || (!next && turn_by > 0))) {
#pragma unroll
            for (int i = 0; i < VE; ++i)
              if (c + i >= 0 && c + i < p.K && (i < VE - turn_by ? !full : !next)) q[c + i] = (int8_t)(mine >> (8 * i));
          }
        }
      }
    }
  } else if constexpr (NORM) {
    // piece after piece, a thread's sixteenth is I8R_PIECES behind its first
    static_assert(16 * G == I8R_PIECES, "the order of the sum");
    const int pieces = (p.K + VE - 1) / VE;
    auto at = [&](const T* v, int c, int off) {
      if (v == nullptr) return make_uint4(0, 0, 0, 0);               // (a row that is not there)
      if (off == 0 || c < off || c - off + 2 * VE > p.K) return i8r_load(v, c, off == 0 ? p.K : 0, p.K);
      return i8r_turn<T>(*reinterpret_cast<const uint4*>(v + c - off), *reinterpret_cast<const uint4*>(v + c - off + VE), off);
    };
    float part[16] = {};
    for (int b = t; b < pieces; b += 16 * G) {
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        if (b + u * G >= pieces) continue;
        float f[VE];
        i8r_unpack<T>(at(x, (b + u * G) * VE, away), f);
        part[u] = __fadd_rn(part[u], i8r_squares(f));
      }
    }
    const float norm = 1.0f / sqrtf(i8r_sum<G>(i8r_join<0, 1, 16>([&](auto u) { return part[decltype(u)::value]; }), red_sum) / (float)p.K + p.eps);
    auto piece = [&](int c, float (&f)[VE]) {
      float g[VE];
      i8r_unpack<T>(at(x, c, away), f);
      i8r_unpack<T>(at(gain, c, (int)(((uintptr_t)gain & 15) / sizeof(T))), g);
#pragma unroll
      for (int i = 0; i < VE; ++i) f[i] = f[i] * norm * g[i];
    };
    uint32_t m = 0;
    for (int b = t; b < pieces; b += G) {
      float f[VE];
      piece(b * VE, f);
#pragma unroll
      for (int i = 0; i < VE; ++i) m = max(m, i8r_bits(f[i]));
    }
    const float amax = i8r_value<float>(i8r_max<G>(m, red_max));
    const Int8Quotient quotient(amax);
    const Int8Pairs pairs(amax);
    int8_t* q = p.q + (size_t)row * p.ldq;
    for (int b = t; b < pieces; b += G) {
      float f[VE];
      uint32_t v[VE];
      piece(b * VE, f);
      if (quotient.ordinary()) {
        i8r_piece<T, false>(pairs, amax, f, v);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = quotient(f[i]);
      }
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (b * VE + i < p.K) q[b * VE + i] = (int8_t)(v[i] & 0xffu);
    }
    for (int i = p.K + t; i < p.ldq; i += G) q[i] = 0;
    if (t == 0) p.s[row] = quotient.scale();
  } else {
    auto element = [&](int i) { return x == nullptr ? 0.0f : to_f(x[i]); };
    uint32_t m = 0;
#pragma unroll 4
    for (int i = t; i < p.K; i += G) m = max(m, i8r_bits(element(i)));
    const Int8Quotient quotient(i8r_value<float>(i8r_max<G>(m, red_max)));
    int8_t* q = p.q + (size_t)row * p.ldq;
#pragma unroll 4
    for (int i = t; i < p.K; i += G) q[i] = (int8_t)(quotient(element(i)) & 0xffu);
    for (int i = p.K + t; i < p.ldq; i += G) q[i] = 0;
    if (t == 0) p.s[row] = quotient.scale();
  }
}

template <typename T, int G, int NV, bool NORM, bool EDGE = false>
static cudaError_t rows_go(const Int8Rows& p, cudaStream_t stream) {
  constexpr int PER = i8r_threads(G) / G;
  return launch_pdl(int8_rows_kernel<T, G, NV, NORM, EDGE>, dim3((unsigned)((p.n + PER - 1) / PER)), dim3(i8r_threads(G)), 0, stream, p);
}

// off the boundary, sixteen pieces a thread (with gains as well that is more than registers hold: not called).  us, before -> so: 32768 x 2047 79 -> 65, 1431 x 26683 81 -> 37
template <typename T, int G, bool NORM>
static cudaError_t rows_edge(const Int8Rows& p, cudaStream_t stream) {
  if constexpr (NORM) return cudaErrorInvalidValue;
  else return rows_go<T, G, 16, false, true>(p, stream);
}

template <typename T, bool NORM>
static int rows_launch(const Int8Rows& p, cudaStream_t stream) {
  constexpr int VE = 16 / sizeof(T);
  const bool whole = p.K % VE == 0 && (p.ldx * (long long)sizeof(T)) % 16 == 0 && ((uintptr_t)p.x & 15) == 0 && p.ldq % VE == 0 && (uintptr_t)p.q % VE == 0 &&
                     ((uintptr_t)p.gain & 15) == 0;
  const int pieces = p.K / VE, spread = (p.K + 2 * VE - 2) / VE;      // pieces of a row: on the boundary; at most, off it
  // few rows: their latency counts, many threads a row; many rows: bytes on their way count, many pieces a thread (us with 256 threads | with one warp: 8192 x 4096 18.2 | 15.3,
  // 8192 x 2048 13.6 | 7.6; 2000 x 4096 5.7 | 6.1)
  const bool few = p.n <= 4 * SMS;
  cudaError_t e;
  if (whole && !few && pieces <= 2 * 8) e = rows_go<T, 8, 2, NORM>(p, stream);
  else if (whole && pieces <= 2 * 32) e = rows_go<T, 32, 2, NORM>(p, stream);
  else if (whole && few && pieces <= 2 * 256) e = rows_go<T, 256, 2, NORM>(p, stream);
  else if (whole && few && pieces <= 8 * 256) e = rows_go<T, 256, 8, NORM>(p, stream);
  else if (whole && pieces <= 8 * 32) e = rows_go<T, 32, 8, NORM>(p, stream);
  else if (whole && pieces <= 16 * 32) e = rows_go<T, 32, 16, NORM>(p, stream);
  else if (whole && pieces <= 8 * 128) e = rows_go<T, 128, 8, NORM>(p, stream);
  else if (whole && pieces <= 16 * 128) e = rows_go<T, 128, 16, NORM>(p, stream);
  else if (whole && pieces <= 16 * 256) e = rows_go<T, 256, 16, NORM>(p, stream);
  else if (!few && spread <= 2 * 8) e = rows_go<T, 8, 2, NORM, true>(p, stream);
  else if (spread <= 2 * 32) e = rows_go<T, 32, 2, NORM, true>(p, stream);
  else if (few && spread <= 2 * 256) e = rows_go<T, 256, 2, NORM, true>(p, stream);
  else if (spread <= 8 * 32) e = rows_go<T, 32, 8, NORM, true>(p, stream);
  else if (!NORM && !few && spread <= 16 * 32) e = rows_edge<T, 32, NORM>(p, stream);
  else if (spread <= 8 * 128) e = rows_go<T, 128, 8, NORM, true>(p, stream);
  else if (spread <= 8 * 256) e = rows_go<T, NORM ? 256 : 128, NORM ? 8 : 16, NORM, true>(p, stream);
  else if (!NORM && spread <= 16 * 256) e = rows_edge<T, 256, NORM>(p, stream);
  else e = rows_go<T, 256, 0, NORM>(p, stream);
  JL_CUDA(e);
  return JL_OK;
}

int int8_rows(const void* x, int dtype, int M, int K, long long ldx, const int* rows, int n, const void* gain, float eps, void* q, int ldq, float* s, int early,
              cudaStream_t stream) {
  Int8Rows p{x, rows, gain, (int8_t*)q, s, M, n, K, ldq, ldx, eps, early};
  JL_DISPATCH_INT8(dtype, return gain != nullptr ? rows_launch<T, true>(p, stream) : rows_launch<T, false>(p, stream));
}

}  // namespace jl

using namespace jl;

extern "C" JL_API int jl_int8_rows(const void* x, int dtype, int M, int K, long long ldx, const int* rows, int n, const void* gain, float eps, void* q, int ldq,
                                   float* s, void* stream) {
  JL_CHECK_ARG(dtype >= DT_BF16 && dtype <= DT_F16, "jl_int8_rows: element type %d", dtype);
  JL_CHECK_ARG(M >= 0 && n >= 0 && n <= I8_MAX_ROWS && K >= 1 && K <= I8_MAX_COLUMNS && ldq >= K && ldq <= I8_MAX_COLUMNS + 16 && (ldx >= K || M <= 1) && (rows != nullptr || n <= M), "jl_int8_rows: %d x %d (pitch %lld) as %d rows of pitch %d", M, K, ldx, n, ldq);
  if (n == 0) return JL_OK;
  return int8_rows(x, dtype, M, K, ldx, rows, n, gain, eps, q, ldq, s, 0, (cudaStream_t)stream);
}
