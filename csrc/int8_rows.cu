// Rows of numbers as int8 values and one scale each: s = amax / 127, q = 127 x / amax rounded to the nearest whole number, ties to even.
//
// Both are what 64 bits would give: s is one rounded quotient, and q is decided exactly.  The quotient is taken in fp32 first (127 / amax once a row, one product an
// element: off by at most 127 * 2^-23 = 1.6e-5); only where it lies within 3e-5 of the middle of two whole numbers are 254 |x| and (2k + 1) amax compared in
// fp64, where both are exact.  A row of zeros has s = 0, a row that holds an infinity or a NaN s = NaN, both with q = 0: what such a row is multiplied with gives
// zeros or NaN.  With gains the row is normed first (RMS, fp32, no rounding in between).
//
// One pass over memory: a row's 16-byte pieces stay in registers between its maximum and its values.  Rows of up to I8R_NARROW columns go eight to a CTA, a warp
// each; longer ones have 256 threads; rows off the 16-byte boundary, and longer ones than registers hold, are read twice, an element a thread.
// Maxima are taken on the bits without their sign, as whole numbers: the order is that of the magnitudes, with infinities and NaN above all of them.
#include "int8.cuh"
#include "jllama_b200.h"

namespace jl {

constexpr int I8R_THREADS = 256;

struct Int8Rows {
  const void* x;
  const int* rows;            // source row of every row of the result, or nullptr: the same
  const void* gain;           // norm first: gains of x's type, or nullptr
  int8_t* q;
  float* s;
  int M, n, K, ldq;           // rows of x, rows of the result, columns, row pitch of q (columns behind K become zeros)
  long long ldx;
  float eps;
  int early;                  // let the next kernel start before this one is done
};

// the magnitude's bits (for 16-bit types the larger of two, in the upper or lower half)
template <typename T> __device__ __forceinline__ uint32_t i8r_bits(T v);
template <> __device__ __forceinline__ uint32_t i8r_bits<float>(float v) { return __float_as_uint(v) & 0x7fffffffu; }
template <> __device__ __forceinline__ uint32_t i8r_bits<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat16_as_ushort(v) & 0x7fffu; }
template <> __device__ __forceinline__ uint32_t i8r_bits<__half>(__half v) { return __half_as_ushort(v) & 0x7fffu; }
template <typename T> __device__ __forceinline__ float i8r_value(uint32_t bits);
template <> __device__ __forceinline__ float i8r_value<float>(uint32_t b) { return __uint_as_float(b); }
template <> __device__ __forceinline__ float i8r_value<__nv_bfloat16>(uint32_t b) { return __uint_as_float(b << 16); }
template <> __device__ __forceinline__ float i8r_value<__half>(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }

template <typename T>
__device__ __forceinline__ void i8r_unpack(const uint4& w, float (&v)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
  } else {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = bf16_lo(u[i]); v[2 * i + 1] = bf16_hi(u[i]);
      }
    }
  }
}

// what a row's elements are multiplied with: x * pre * inv = 127 x / amax.  pre lifts rows so small that 127 / amax would overflow.
struct Int8Quotient {
  float pre, inv, amax;
  __device__ __forceinline__ explicit Int8Quotient(float a) {
    amax = a;
    pre = a < 0x1p-60f ? 0x1p64f : 1.0f;
    inv = a > 0.0f && a <= 3.402823466e38f ? __fdiv_rn(127.0f, a * pre) : 0.0f;
  }
  __device__ __forceinline__ float scale() const { return amax <= 3.402823466e38f ? __fdiv_rn(amax, 127.0f) : __int_as_float(0x7fc00000); }
  // the value as the low byte of the result
  __device__ __forceinline__ uint32_t operator()(float x) const {
    const float t = x * pre * inv;
    const float magic = t + 12582912.0f;                         // 1.5 * 2^23: the nearest whole number, ties to even, in the low bits
    uint32_t q = __float_as_uint(magic);
    if (fabsf(t - (magic - 12582912.0f)) > 0.49997f) {
      const int k = (int)fabsf(t);                               // between k and k + 1, near the middle
      const double a = 254.0 * (double)fabsf(x), b = (2.0 * k + 1.0) * (double)amax;
      const int r = a > b ? k + 1 : a < b ? k : k + (k & 1);
      q = (uint32_t)(x < 0.0f ? -r : r);
    }
    return inv == 0.0f ? 0u : q;                                 // (inf * 0 and NaN go nowhere)
  }
};
__device__ __forceinline__ uint32_t i8r_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <int G>
__device__ __forceinline__ uint32_t i8r_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (G == 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < G / 32; ++i) v = max(v, red[i]);
  return v;
}
template <int G>
__device__ __forceinline__ float i8r_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (G == 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int i = 0; i < G / 32; ++i) v += red[i];
  return v;
}

// G threads a row, up to NV 16-byte pieces a thread; NV = 0: element by element, any row
template <typename T, int G, int NV, bool NORM>
__global__ void __launch_bounds__(I8R_THREADS) int8_rows_kernel(const Int8Rows p) {
  __shared__ uint32_t red[2 * I8R_THREADS / 32];
  pdl_wait();
  if (p.early) pdl_launch_dependents();
  const int t = threadIdx.x % G, row = blockIdx.x * (I8R_THREADS / G) + threadIdx.x / G;
  if (row >= p.n) return;                                        // (whole groups)
  const int src = p.rows != nullptr ? p.rows[row] : row;
  const bool there = src >= 0 && src < p.M;                      // a row that is not there is zeros
  const T* x = reinterpret_cast<const T*>(p.x) + (there ? (long long)src * p.ldx : 0);
  const T* gain = reinterpret_cast<const T*>(p.gain);
  int8_t* q = p.q + (size_t)row * p.ldq;
  constexpr int VE = 16 / sizeof(T);
  uint32_t* red_max = red;
  float* red_sum = reinterpret_cast<float*>(red + I8R_THREADS / 32);
  float norm = 1.0f;
  if constexpr (NV > 0) {
    const int pieces = p.K / VE;
    uint4 w[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) w[v] = there && t + v * G < pieces ? reinterpret_cast<const uint4*>(x)[t + v * G] : make_uint4(0, 0, 0, 0);
    uint32_t m = 0;
    if constexpr (NORM) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float f[VE];
        i8r_unpack<T>(w[v], f);
#pragma unroll
        for (int i = 0; i < VE; ++i) sum = fmaf(f[i], f[i], sum);
      }
      norm = 1.0f / sqrtf(i8r_sum<G>(sum, red_sum) / (float)p.K + p.eps);
    }
    auto element = [&](float x0, float g) { return NORM ? x0 * norm * g : x0; };
    auto gains = [&](int v, float (&g)[VE]) {
      if constexpr (NORM) {
        if (t + v * G < pieces) i8r_unpack<T>(reinterpret_cast<const uint4*>(gain)[t + v * G], g);
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
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (t + v * G >= pieces) break;
      float f[VE], g[VE] = {};
      i8r_unpack<T>(w[v], f);
      gains(v, g);
      uint32_t b[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) b[i] = quotient(element(f[i], g[i]));
      if constexpr (VE == 8) reinterpret_cast<uint2*>(q)[t + v * G] = make_uint2(i8r_pack4(b[0], b[1], b[2], b[3]), i8r_pack4(b[4], b[5], b[6], b[7]));
      else reinterpret_cast<uint32_t*>(q)[t + v * G] = i8r_pack4(b[0], b[1], b[2], b[3]);
    }
    for (int i = p.K + t; i < p.ldq; i += G) q[i] = 0;
    if (t == 0) p.s[row] = quotient.scale();
  } else {
    if constexpr (NORM) {
      float sum = 0.0f;
      for (int i = t; i < p.K; i += G) { const float f = there ? to_f(x[i]) : 0.0f; sum = fmaf(f, f, sum); }
      norm = 1.0f / sqrtf(i8r_sum<G>(sum, red_sum) / (float)p.K + p.eps);
    }
    auto element = [&](int i) { return !there ? 0.0f : NORM ? to_f(x[i]) * norm * to_f(gain[i]) : to_f(x[i]); };
    uint32_t m = 0;
#pragma unroll 4
    for (int i = t; i < p.K; i += G) m = max(m, i8r_bits(element(i)));
    const Int8Quotient quotient(i8r_value<float>(i8r_max<G>(m, red_max)));
#pragma unroll 4
    for (int i = t; i < p.K; i += G) q[i] = (int8_t)(quotient(element(i)) & 0xffu);
    for (int i = p.K + t; i < p.ldq; i += G) q[i] = 0;
    if (t == 0) p.s[row] = quotient.scale();
  }
}

template <typename T, bool NORM>
static int rows_launch(const Int8Rows& p, cudaStream_t stream) {
  constexpr int VE = 16 / sizeof(T);
  const bool whole = p.K % VE == 0 && (p.ldx * (long long)sizeof(T)) % 16 == 0 && ((uintptr_t)p.x & 15) == 0 && p.ldq % VE == 0 && (uintptr_t)p.q % VE == 0 &&
                     ((uintptr_t)p.gain & 15) == 0;
  const int pieces = p.K / VE;
  auto go = [&](auto kernel, int group) {
    const int per = I8R_THREADS / group;
    return launch_pdl(kernel, dim3((unsigned)((p.n + per - 1) / per)), dim3(I8R_THREADS), 0, stream, p);
  };
  cudaError_t e;
  if (whole && pieces <= 2 * 32) e = go(int8_rows_kernel<T, 32, 2, NORM>, 32);
  else if (whole && pieces <= 8 * 32) e = go(int8_rows_kernel<T, 32, 8, NORM>, 32);
  else if (whole && pieces <= 2 * 256) e = go(int8_rows_kernel<T, 256, 2, NORM>, 256);
  else if (whole && pieces <= 4 * 256) e = go(int8_rows_kernel<T, 256, 4, NORM>, 256);
  else if (whole && pieces <= 8 * 256) e = go(int8_rows_kernel<T, 256, 8, NORM>, 256);
  else if (whole && pieces <= 16 * 256) e = go(int8_rows_kernel<T, 256, 16, NORM>, 256);
  else if (p.K <= 512) e = go(int8_rows_kernel<T, 32, 0, NORM>, 32);
  else e = go(int8_rows_kernel<T, 256, 0, NORM>, 256);
  JL_CUDA(e);
  return JL_OK;
}

int int8_rows(const void* x, int dtype, int M, int K, long long ldx, const int* rows, int n, const void* gain, float eps, void* q, int ldq, float* s, bool early,
              cudaStream_t stream) {
  Int8Rows p{x, rows, gain, (int8_t*)q, s, M, n, K, ldq, ldx, eps, early};
  JL_DISPATCH_INT8(dtype, return gain != nullptr ? rows_launch<T, true>(p, stream) : rows_launch<T, false>(p, stream));
}

}  // namespace jl

using namespace jl;

extern "C" JL_API int jl_int8_rows(const void* x, int dtype, int M, int K, long long ldx, const int* rows, int n, const void* gain, float eps, void* q, int ldq,
                                   float* s, void* stream) {
  JL_CHECK_ARG(dtype >= DT_BF16 && dtype <= DT_F16, "jl_int8_rows: element type %d", dtype);
  JL_CHECK_ARG(M >= 0 && n >= 0 && K >= 1 && ldq >= K && (ldx >= K || M <= 1) && (rows != nullptr || n <= M), "jl_int8_rows: %d x %d (pitch %lld) as %d rows of pitch %d", M, K, ldx, n, ldq);
  if (n == 0) return JL_OK;
  return int8_rows(x, dtype, M, K, ldx, rows, n, gain, eps, q, ldq, s, false, (cudaStream_t)stream);
}
