// What the kernels of 8-bit integer layers share: element types, the store of finished results, the way a list of tiles covers the rows of every expert.
//
// A layer is y[m, n] = sx[m] sw[n] sum_k qx[m, k] qw[n, k]: int8 values, one fp32 scale per row of either side, sums in int32 (exact: |q| <= 127 and K <= 131072
// keep them below 2^31), then fp32 until the one rounding to the result's type.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "seq_types.cuh"

namespace jl {

enum { DT_F16 = 2 };                                             // beside DT_BF16 and DT_F32
enum { I8_PLAIN = 0, I8_RESIDUAL = 1, I8_GATED = 2, I8_RELU2 = 3 };      // result; result + residual; silu(y[2j]) y[2j+1]; relu(y)^2
constexpr int I8_MAX_K = 131072;
constexpr int I8_MAX_EXPERTS = 1024;
constexpr int I8_MAX_ROWS = 1 << 30;
constexpr int I8_MAX_COLUMNS = 1 << 30;      // of rows alone; columns and a block's threads behind them stay whole numbers of 32 bits

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

#define JL_DISPATCH_INT8(dt, ...)                                        \
  do {                                                                   \
    if ((dt) == jl::DT_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }   \
    else if ((dt) == jl::DT_F32) { using T = float; __VA_ARGS__; }       \
    else { using T = __half; __VA_ARGS__; }                              \
  } while (0)

// the magnitude's bits, and the magnitude that they are
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
  __device__ __forceinline__ bool ordinary() const { return amax >= 0x1p-60f && amax <= 3.402823466e38f; }      // (not zero, not tiny, all of them numbers)
  __device__ __forceinline__ float scale() const { return amax <= 3.402823466e38f ? __fdiv_rn(amax, 127.0f) : __int_as_float(0x7fc00000); }
  // any row: the value as the low byte of the result
  __device__ __forceinline__ uint32_t operator()(float x) const {
    const float t = x * pre * inv;
    const float magic = t + 12582912.0f;                         // 1.5 * 2^23: the nearest whole number, ties to even, in the low bits
    uint32_t q = __float_as_uint(magic);
    if (fabsf(t - (magic - 12582912.0f)) > 0.49997f) {      // (off by at most 1.6e-5)
      const int k = (int)fabsf(t);                               // between k and k + 1, near the middle
      const double a = 254.0 * (double)fabsf(x), b = (2.0 * k + 1.0) * (double)amax;
      const int r = a > b ? k + 1 : a < b ? k : k + (k & 1);
      q = (uint32_t)(x < 0.0f ? -r : r);
    }
    return inv == 0.0f ? 0u : q;                                 // (inf * 0 and NaN go nowhere)
  }
};

// Ordinary rows, two elements at a time (packed fp32).  With X = 127 x and a = amax (both by 2^-8, which keeps X finite) the quotient is t0 = X * (1 / a), corrected once by what
// it leaves (Markstein, 1990): t = t0 + (X - t0 a) (1 / a).  t0 is off by a share d of a few 2^-24, the remainder is taken with one rounding, so t before its own rounding is off by d 2^-24 or so:
//   * a quotient on the middle k + 1/2, which fp32 holds, comes out as that, and the sum with 1.5 * 2^23 rounds it to the even side;
//   * rounding t does not carry it over a middle, and onto one only from less than 2^-24 t away.  With x and amax of p bits, exponents e apart, the nearest quotient beside a
//     middle is 2^(e - p - 1) away, and 2^-24 t is at most 2^(e - 16): never for the 16-bit types (p = 8, 11).
// fp32 rows can come that near: quotients within I8R_NEAR of a middle are settled.  (16-bit rows meet middles often, amax / 2 is one at every scale: a quarter of all groups
// of 256 elements.  Settling those too took 313 us for 8192 x 14336, most of it for instructions that were not in the cache.)
constexpr float I8R_NEAR = 0.49999f;      // (a step of fp32 below 128 is 7.6e-6)
struct Int8Pairs {
  uint64_t a, inv;            // -a and 1 / a, twice
  __device__ __forceinline__ explicit Int8Pairs(float amax) {
    const float lo = amax * 0x1p-8f, r = __fdiv_rn(1.0f, lo);
    asm("mov.b64 %0, {%1, %1};" : "=l"(a) : "f"(-lo));
    asm("mov.b64 %0, {%1, %1};" : "=l"(inv) : "f"(r));
  }
  // the whole numbers in the low bytes; `off`: how far the worst quotient so far lies from a whole number
  template <bool OFF>
  __device__ __forceinline__ void get(float x0, float x1, uint32_t& q0, uint32_t& q1, float& off) const {
    uint64_t x, t, e, m;
    const uint64_t c = 0x3efe00003efe0000ull, magic = 0x4b4000004b400000ull;      // 127 / 256 and 1.5 * 2^23, twice
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(x0), "f"(x1));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(x), "l"(c));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t) : "l"(x), "l"(inv));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(e) : "l"(t), "l"(a), "l"(x));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t) : "l"(e), "l"(inv), "l"(t));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(m) : "l"(t), "l"(magic));
    asm("mov.b64 {%0, %1}, %2;" : "=r"(q0), "=r"(q1) : "l"(m));
    if constexpr (OFF) {
      float t0, t1;
      asm("mov.b64 {%0, %1}, %2;" : "=f"(t0), "=f"(t1) : "l"(t));
      off = fmaxf(off, fmaxf(fabsf(t0 - (__uint_as_float(q0) - 12582912.0f)), fabsf(t1 - (__uint_as_float(q1) - 12582912.0f))));
    }
  }
};
// The whole number that a rounded quotient of x gave, or the one beside it, exactly: r against 127 x - r amax.  Both products are taken with what their rounding
// left; near a middle the differences of the large parts are exact, so is that of the small ones, and the last sum has the right sign.
static __device__ __noinline__ uint4 i8r_settle4(float4 v, uint4 bits, float amax) {
  const float a = amax * 0x1p-8f, h = 0.5f * a;
  const float x[4] = {v.x, v.y, v.z, v.w};
  uint32_t b[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    float r = __uint_as_float(b[i]) - 12582912.0f;
    const float X = x[i] * 0x1p-8f, hi = 127.0f * X, lo = fmaf(127.0f, X, -hi), hi2 = r * a, lo2 = fmaf(r, a, -hi2);
    const float d = hi - hi2, e = lo - lo2, over = (d - h) + e, under = (d + h) + e;
    const bool odd = b[i] & 1;
    r += over > 0.0f || (over == 0.0f && odd) ? 1.0f : under < 0.0f || (under == 0.0f && odd) ? -1.0f : 0.0f;
    b[i] = __float_as_uint(r + 12582912.0f);
  }
  return make_uint4(b[0], b[1], b[2], b[3]);
}
// a piece of an ordinary row.  EXACT: x is what the row holds (rows behind a norm are rounded already)
template <typename T, bool EXACT>
__device__ __forceinline__ void i8r_piece(const Int8Pairs& pairs, float amax, const float (&f)[16 / sizeof(T)], uint32_t (&b)[16 / sizeof(T)]) {
  constexpr int VE = 16 / sizeof(T);
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < VE; i += 2) pairs.get<EXACT && VE == 4>(f[i], f[i + 1], b[i], b[i + 1], off);
  if constexpr (EXACT && VE == 4) {
    if (off > I8R_NEAR) {
      const uint4 s = i8r_settle4(make_float4(f[0], f[1], f[2], f[3]), make_uint4(b[0], b[1], b[2], b[3]), amax);
      b[0] = s.x; b[1] = s.y; b[2] = s.z; b[3] = s.w;
    }
  }
}
// The sum of squares of a row that is normed first has one order, whatever kernel takes the row, so that its values and scale do not depend on the rows beside it.  The squares of a
// 16-byte piece, one that begins at a column that is a multiple of its elements, are added in turn; pieces I8R_PIECES apart are added in rising order; of the I8R_PIECES sums the upper half is added
// to the lower one, half by half.  A piece that is not there adds a zero and changes nothing.  The upper bits of a piece's number are those of a thread's own pieces (t + v G), then the warp's, then the lane's.
constexpr int I8R_PIECES = 4096;
// leaves FIRST, FIRST + STEP, .. below N joined so
template <int FIRST, int STEP, int N, typename F>
__device__ __forceinline__ float i8r_join(const F& leaf) {
  if constexpr (STEP == N) return leaf(std::integral_constant<int, FIRST>{});
  else return __fadd_rn(i8r_join<FIRST, 2 * STEP, N>(leaf), i8r_join<FIRST + STEP, 2 * STEP, N>(leaf));
}
template <int VE>
__device__ __forceinline__ float i8r_squares(const float (&f)[VE]) {
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < VE; ++e) s = fmaf(f[e], f[e], s);
  return s;
}

__device__ __forceinline__ uint32_t i8r_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Dynamic shared memory that a kernel may ask for (set once per device, to one value: calls at the same time do not lower it for one another)
template <auto KERNEL, int BYTES = 227 * 1024>
static cudaError_t i8_room() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (bit & done.load(std::memory_order_relaxed)) return cudaSuccess;
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

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
// silu(g) u.  The quotient is the product with an approximate reciprocal (two units in the last place): a true one branches, and values then wait for one another.  From
// 1 + exp(-g) = 2^126 on the reciprocal is 0 and so is the result, where g e^g u is of less than 2^-119 |u|
__device__ __forceinline__ float i8_gate(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }

// relu(y)^2; a NaN stays one
__device__ __forceinline__ float i8_relu2(float y) {
  const float r = y <= 0.0f ? 0.0f : y;
  return r * r;
}

// Four neighbouring residuals, asked for ahead of i8_finish4 (no load passes a store to what may be the same buffer) and held as they are in memory where KIND, the type, is known.
template <int KIND>
struct Int8Four {
  static constexpr bool packed = KIND == DT_BF16 || KIND == DT_F16;
  std::conditional_t<packed, uint2, float4> v;
  __device__ __forceinline__ void load(const Int8Out& o, int row, int f0) {
    if (f0 >= o.N) return;
    const size_t at = (size_t)row * o.ldo + f0;
    const int kind = KIND >= 0 ? KIND : o.kind;
    if constexpr (packed) {
      const uint16_t* r = reinterpret_cast<const uint16_t*>(o.residual) + at;
      if (o.wide) { v = *reinterpret_cast<const uint2*>(r); return; }
      uint32_t e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = f0 + i < o.N ? r[i] : 0u;
      v = make_uint2(e[0] | e[1] << 16, e[2] | e[3] << 16);
    } else if (o.wide && kind == DT_F32) {
      v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(o.residual) + at);
    } else if (o.wide) {
      const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(o.residual) + at);
      const float2 a = i8_unpack(kind, w.x), b = i8_unpack(kind, w.y);
      v = make_float4(a.x, a.y, b.x, b.y);
    } else {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = f0 + i < o.N ? i8_load(o.residual, kind, at + i) : 0.0f;
      v = make_float4(e[0], e[1], e[2], e[3]);
    }
  }
  __device__ __forceinline__ float4 floats() const {
    if constexpr (packed) {
      const float2 a = i8_unpack(KIND, v.x), b = i8_unpack(KIND, v.y);
      return make_float4(a.x, a.y, b.x, b.y);
    } else {
      return v;
    }
  }
};
// KIND: the result's type where the kernel is one of it (what is finished runs once a launch from cold instructions: fewer are faster), or -1.
// Finishes and stores features f0 .. f0 + 3 (f0 a multiple of four) of a row of the result from their sums
template <int MODE, int KIND = -1>
__device__ __forceinline__ void i8_finish4(const Int8Out& o, int row, int f0, const int (&acc)[4], float sx, const float (&sw)[4], const Int8Four<KIND>& residual) {
  const int kind = KIND >= 0 ? KIND : o.kind;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __int2float_rn(acc[i]) * sx * sw[i];
  if constexpr (MODE == I8_GATED) {
    const float a = i8_gate(y[0], y[1]), b = i8_gate(y[2], y[3]);
    const size_t at = (size_t)row * o.ldo + f0 / 2;
    if (o.wide && f0 + 3 < o.N) {
      if (kind == DT_F32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(o.out) + at) = make_float2(a, b);
      else *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(o.out) + at) = i8_pack(kind, a, b);
      return;
    }
    if (f0 < o.N) i8_store(o.out, kind, at, a);
    if (f0 + 2 < o.N) i8_store(o.out, kind, at + 1, b);
    return;
  }
  if constexpr (MODE == I8_RELU2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = i8_relu2(y[i]);
  }
  const size_t at = (size_t)row * o.ldo + f0;
  if constexpr (MODE == I8_RESIDUAL) {
    const float4 r = residual.floats();       // never fused with the scale's product: a row's bits do not depend on the kernel
    y[0] = __fadd_rn(y[0], r.x); y[1] = __fadd_rn(y[1], r.y); y[2] = __fadd_rn(y[2], r.z); y[3] = __fadd_rn(y[3], r.w);
  }
  if (o.wide) {
    if (kind == DT_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(o.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
    else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(o.out) + at) = make_uint2(i8_pack(kind, y[0], y[1]), i8_pack(kind, y[2], y[3]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (f0 + i < o.N) i8_store(o.out, kind, at + i, y[i]);
}

// The work of a launch as a list: `chunks` pieces of at most `chunk` rows of every expert times `cols` tiles of features; a tile's pieces are neighbours, since they
// share its weights.  Without experts there is one, with all rows.
struct Int8Work {
  const int* offsets;         // [experts + 1]: first row of every expert, and behind the last; or nullptr
  int experts, rows, chunk, cols;
};
struct Int8Tile { int expert, col, row0, rows; };

// first row of expert e, whatever the offsets say: never outside the rows there are.  (Read from L2: the caller may not have waited for the kernel ahead, which began
// when those before it were done.)
__device__ __forceinline__ int i8_offset(const Int8Work& w, int e) { return min(max(__ldcg(w.offsets + e), 0), w.rows); }

// table[e]: tiles ahead of expert e (experts + 1 of them), table[experts + 1 + e]: its first row (experts + 1).  By one warp.
__device__ __forceinline__ void i8_list(const Int8Work& w, int* table) {
  const int lane = threadIdx.x & 31, E = w.experts;
  if (w.offsets == nullptr) {
    if (lane == 0) { table[0] = 0; table[1] = (w.rows + w.chunk - 1) / w.chunk * w.cols; table[2] = 0; table[3] = w.rows; }
    return;
  }
  int ahead = 0;
  for (int e0 = 0; e0 < E; e0 += 128) {             // four neighbours a lane: their offsets come at once
    const int e = e0 + 4 * lane;
    int at[5], tiles[4];
#pragma unroll
    for (int i = 0; i < 5; ++i) at[i] = i8_offset(w, min(e + i, E));
    int incl = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      tiles[i] = (max(at[i + 1] - at[i], 0) + w.chunk - 1) / w.chunk * w.cols;
      incl += tiles[i];
    }
    const int mine = incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    int before = ahead + incl - mine;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (e + i < E) { table[e + i] = before; table[E + 1 + e + i] = at[i]; }
      before += tiles[i];
    }
    ahead += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) { table[E] = ahead; table[2 * E + 1] = i8_offset(w, E); }
}

// walks the list in rising order
struct Int8Walk {
  int e = 0;
  __device__ __forceinline__ Int8Tile at(const Int8Work& w, const int* table, int t) {
    // the last expert whose tiles begin at or ahead of t: steps that double, then halve (128 experts, one by one: 2 us)
    int step = 1;
    for (; e + step < w.experts && t >= table[e + step]; step *= 2) e += step;
    for (; step > 0; step /= 2)
      if (e + step < w.experts && t >= table[e + step]) e += step;
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
// pieces of `chunk` rows, at most: every expert that has rows may have one that is not full
inline long long i8_pieces(const Int8Work& w, int chunk) {
  if (w.offsets == nullptr) return ((long long)w.rows + chunk - 1) / chunk;
  return w.rows <= w.experts ? w.rows : w.experts + ((long long)w.rows - w.experts) / chunk;
}

}  // namespace jl
