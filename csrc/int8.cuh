// What the kernels of 8-bit integer layers share: element types, the store of finished results, the way a list of tiles covers the rows of every expert.
//
// A layer is y[m, n] = sx[m] sw[n] sum_k qx[m, k] qw[n, k]: int8 values, one fp32 scale per row of either side, sums in int32 (exact: |q| <= 127 and K <= 131072
// keep them below 2^31), then fp32 until the one rounding to the result's type.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "seq_types.cuh"

namespace jl {

enum { DT_F16 = 2 };                                             // beside DT_BF16 and DT_F32
enum { I8_PLAIN = 0, I8_RESIDUAL = 1, I8_GATED = 2 };            // result; result + residual; silu(y[2j]) y[2j+1]
constexpr int I8_MAX_K = 131072;
constexpr int I8_MAX_EXPERTS = 1024;

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

#define JL_DISPATCH_INT8(dt, ...)                                        \
  do {                                                                   \
    if ((dt) == jl::DT_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }   \
    else if ((dt) == jl::DT_F32) { using T = float; __VA_ARGS__; }       \
    else { using T = __half; __VA_ARGS__; }                              \
  } while (0)

// Result, residual and scales of a product
struct Int8Out {
  void* out;
  const void* residual;       // I8_RESIDUAL: [rows, N] of the result's type
  const float* xs;            // scale of every row
  const float* ws;            // scale of every feature (of every expert)
  int kind, N, ldo, wide;     // type of the result; features; row pitch; wide: four neighbouring features are one access
};

__device__ __forceinline__ float i8_load(const void* p, int kind, size_t i) {
  if (kind == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (kind == DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void i8_store(void* p, int kind, size_t i, float v) {
  if (kind == DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (kind == DT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ uint32_t i8_pack(int kind, float a, float b) {
  if (kind == DT_BF16) return pack_bf16(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 i8_unpack(int kind, uint32_t w) {
  if (kind == DT_BF16) return make_float2(bf16_lo(w), bf16_hi(w));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float i8_gate(float g, float u) { return g * sigmoid_f(g) * u; }

// four neighbouring residuals (index of the first one: a multiple of four where `wide`)
__device__ __forceinline__ void i8_residual4(const Int8Out& o, size_t at, int f0, float (&r)[4]) {
  if (o.wide) {
    if (o.kind == DT_F32) {
      load4(reinterpret_cast<const float*>(o.residual) + at, r);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(o.residual) + at);
      const float2 a = i8_unpack(o.kind, w.x), b = i8_unpack(o.kind, w.y);
      r[0] = a.x; r[1] = a.y; r[2] = b.x; r[3] = b.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = f0 + i < o.N ? i8_load(o.residual, o.kind, at + i) : 0.0f;
}

// finishes and stores features f0 .. f0 + 3 (f0 a multiple of four) of a row of the result from their sums
template <int MODE>
__device__ __forceinline__ void i8_finish4(const Int8Out& o, int row, int f0, const int (&acc)[4], float sx, const float (&sw)[4]) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __int2float_rn(acc[i]) * sx * sw[i];
  if constexpr (MODE == I8_GATED) {
    const float a = i8_gate(y[0], y[1]), b = i8_gate(y[2], y[3]);
    const size_t at = (size_t)row * o.ldo + f0 / 2;
    if (o.wide && f0 + 3 < o.N) {
      if (o.kind == DT_F32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(o.out) + at) = make_float2(a, b);
      else *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(o.out) + at) = i8_pack(o.kind, a, b);
      return;
    }
    if (f0 < o.N) i8_store(o.out, o.kind, at, a);
    if (f0 + 2 < o.N) i8_store(o.out, o.kind, at + 1, b);
    return;
  }
  const size_t at = (size_t)row * o.ldo + f0;
  if constexpr (MODE == I8_RESIDUAL) {
    float r[4];
    i8_residual4(o, at, f0, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] += r[i];
  }
  if (o.wide) {
    if (o.kind == DT_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(o.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
    else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(o.out) + at) = make_uint2(i8_pack(o.kind, y[0], y[1]), i8_pack(o.kind, y[2], y[3]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (f0 + i < o.N) i8_store(o.out, o.kind, at + i, y[i]);
}

// The work of a launch as a list: `chunks` pieces of at most `chunk` rows of every expert times `cols` tiles of features; a tile's pieces are neighbours, since they
// share its weights.  Without experts there is one, with all rows.
struct Int8Work {
  const int* offsets;         // [experts + 1]: first row of every expert, and behind the last; or nullptr
  int experts, rows, chunk, cols;
};
struct Int8Tile { int expert, col, row0, rows; };

// first row of expert e, whatever the offsets say: never outside the rows there are
__device__ __forceinline__ int i8_offset(const Int8Work& w, int e) { return min(max(w.offsets[e], 0), w.rows); }

// table[e]: tiles ahead of expert e (experts + 1 of them), table[experts + 1 + e]: its first row (experts + 1).  By one warp.
__device__ __forceinline__ void i8_list(const Int8Work& w, int* table) {
  const int lane = threadIdx.x & 31, E = w.experts;
  if (w.offsets == nullptr) {
    if (lane == 0) { table[0] = 0; table[1] = (w.rows + w.chunk - 1) / w.chunk * w.cols; table[2] = 0; table[3] = w.rows; }
    return;
  }
  int ahead = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    int a = 0, n = 0;
    if (e < E) {
      a = i8_offset(w, e);
      n = max(i8_offset(w, e + 1) - a, 0);
    }
    const int mine = (n + w.chunk - 1) / w.chunk * w.cols;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (e < E) { table[e] = ahead + incl - mine; table[E + 1 + e] = a; }
    ahead += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) { table[E] = ahead; table[2 * E + 1] = i8_offset(w, E); }
}

// walks the list in rising order
struct Int8Walk {
  int e = 0;
  __device__ __forceinline__ Int8Tile at(const Int8Work& w, const int* table, int t) {
    while (t >= table[e + 1]) ++e;
    const int row = table[w.experts + 1 + e], end = table[w.experts + 2 + e];
    const int pieces = (end - row + w.chunk - 1) / w.chunk, i = t - table[e];
    Int8Tile tile;
    tile.expert = e;
    tile.col = i / pieces;
    tile.row0 = row + i % pieces * w.chunk;
    tile.rows = min(w.chunk, end - tile.row0);
    return tile;
  }
};
__host__ __device__ constexpr int i8_table_ints(int experts) { return 2 * experts + 2; }

}  // namespace jl
