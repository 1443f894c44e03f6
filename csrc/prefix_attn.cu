// Attention of a batch whose rows share keys: a prompt with several answers, a document with many questions.
//
//   out(b, s, h) = softmax_j (q · k_j / sqrt(d)) v_j   over the keys [prefix_pad, prefix_len) of the row's group, the same for all its rows, and the
//                  row's own keys [pad_left, slot of the query]
//
// The shared keys are read once for all rows: the queries of a group, every row's tokens and the G query heads of a key head, are the rows of one
// matrix [rows · S · G, d] per (group, key head), cut into tiles of 128 for tcgen05.  With running statistics a softmax over two sets of keys
// is a join of two triples (reference exponent m, sum l, weighted values o):  M = max(m1, m2),  o = o1 2^(m1 - M) + o2 2^(m2 - M),  l likewise.
//   * one token per row (jl_decode_attn_prefix): one launch in which some CTAs take the shared keys, tiles of queries by splits of the keys, and others the
//     rows' own keys, a warp per (row, key head), appending the new one; all leave partial triples in fp32, and a second, small launch joins them; with up to
//     eight queries of a (group, key head), warps take the shared keys too;
//   * S tokens per row (jl_prefill_attn_prefix): the same for the shared keys, then a second launch over every row's own keys, causal, in tiles or, a few tokens, by
//     warps, and the join; or, where a row's queries fill tiles by themselves, one launch over both sets of keys, tile after tile, whole or in splits that the join
//     puts together.
//
// One CTA owns a tile of 128 queries of one key head, as in flash_prefill.cu: a warp asks for K and V tiles of 64 keys (TMA, 128-byte swizzle), a warp
// issues S = Q·Kᵀ into one of two score tiles in TMEM and O += P·V with P read from TMEM, four warps hold one query row per thread: one pass over 64
// scores in registers, exponentials in base 2 against a reference that is raised only when it has grown by 2^8.
// Queries go to shared memory by hand: rows of different tokens and heads follow each other in a tile, and the one-token form rotates them on the way.
// A rotated query is kept as two bfloat16 numbers, hi + lo (two products into the same scores): rounded to one, a score of size s would be off by
// s 2^-8 and the result by as much again as its own rounding.  Probabilities of a step are hi + lo too, as in decode_attn_fused.cu, so that a row's result
// has the same bits however many rows share the keys.  Those of prompts are where a launch has one tile of queries and the products have time to spare; with
// more they are rounded to bfloat16 (2^-8 of each weight, sums in fp32), as flash_prefill.cu rounds those of the same rows written out.
// Slots that hold no key may hold anything: their scores are masked, and their value rows are cleared in shared memory, because a weight of zero
// times a NaN is a NaN.
//
// One B200, us a call in a graph of ten, by itself: one token, 16 rows x 32 heads over 8 of keys, 2048 shared 12.7; 96 rows, 32768 shared and 500 own each 122 (860 TFLOP/s with the
// second products of queries and probabilities, 2.7 TB/s beside them); 4 x 16 rows, 3501 shared and 701 own 44 (5.5 TB/s).  Prompts: 2 x 2048 tokens over 16384 1065 (1080 TFLOP/s; a
// single launch of its own 906 and 1290: the power cap), 8 x 333 over 1500 68 (1110), 16 x 48 over 8192 111 (920).  What bounds them: products of small width
// (a 128 x 64 tile of scores reads its queries from shared memory, 384 cycles for 256 of products) and the exponentials, half of the special-function
// unit's rate with a quarter of them on the FMA units; in short calls the chain launch, queries, scores, last rows, join.
#include <atomic>

#include "jllama_b200.h"
#include "tcgen05.cuh"

namespace jl {

constexpr int PX_BM = 128, PX_BN = 64, PX_THREADS = 352;
constexpr float PX_RESCALE = 8.0f;                                 // log2 units

// The CTAs of a step that take the rows' own keys: WARPS independent warps with a ring of STAGES blocks of KPI keys and values each.
template <int HD> struct PxOwn {
  static constexpr int WARPS = 8, STAGES = 3, HALVES = HD / 64;
  static constexpr int KPI = HD == 128 ? 16 : 32;                  // 8 KB of keys and values at either width
  static constexpr uint32_t BOX = KPI * 128, STAGE = 2 * HALVES * BOX, RING = STAGES * STAGE;
  static constexpr uint32_t QT = 16 * HD * 2;                      // a unit's queries: 8 rows of high parts, 8 of low ones
  static constexpr uint32_t SMEM = WARPS * (RING + QT) + 1024;
};

// How a CTA works.  PX_PAIR: two tiles of queries, each with its own softmax warps, over the same keys.  PX_TURNS: one tile whose keys the two sets of softmax warps
// take in turn.  PX_SOLO: one tile, one set, half an SM (its way in and out falls into the other half's work).
constexpr int PX_TURNS = 0, PX_PAIR = 1, PX_SOLO = 2;

template <int HD, bool ROTATE, int MODE> struct PxTile {
  static constexpr bool PAIR = MODE != PX_TURNS, SOLO = MODE == PX_SOLO, JOINT = MODE == PX_PAIR;        // PAIR: a set walks all tiles with queries of its own
  static constexpr int HALVES = HD / 64;
  static constexpr uint32_t Q_HALF = PX_BM * 128, Q = HALVES * Q_HALF;       // bytes of a tile of queries (hi or lo)
  static constexpr int NQ = ROTATE ? 2 : 1;                                  // hi, lo
  static constexpr uint32_t QS = (JOINT ? 2 : 1) * NQ * Q;
  static constexpr int ROWS = (JOINT ? 2 : 1) * PX_BM, SETS = SOLO ? 1 : 2, THREADS = SOLO ? 192 : PX_THREADS;      // (two warps and four for each set; one more for two)
  static constexpr uint32_t KV_HALF = PX_BN * 128, KV = HALVES * KV_HALF;    // 64 columns of a tile of keys or values, all of them
  // A slot of the ring holds both (JOINT: one wait and one release per tile, the warps that issue products have none to spare), or keys and values in turn (the keys'
  // place is free again as soon as their scores are there: with both in one slot the four tiles that the two sets work on held the whole ring, and the keys of 48
  // rows x 32 heads came in at 29 GB/s per SM)
  static constexpr uint32_t SLOT = (JOINT ? 2 : 1) * KV;
  static constexpr uint32_t SMALL = 512 + (PAIR ? 0 : 2048);                 // barriers, the address of the TMEM columns; (m, l) of 2 x 128 rows
  static constexpr uint32_t MOST = (SOLO ? 113 : 227) * 1024;
  static constexpr int FIT = (int)((MOST - 1024 - SMALL - QS) / SLOT);
  static constexpr int SLOTS = FIT < 16 ? FIT : 16;
  static constexpr uint32_t NEED = QS + SLOTS * SLOT + SMALL + 1024;         // (1024: alignment of the base)
  static constexpr uint32_t SMEM = ROTATE && NEED < PxOwn<HD>::SMEM ? PxOwn<HD>::SMEM : NEED;
  static_assert(SLOTS >= (SOLO ? 4 : (JOINT ? 3 : 8)) && SMEM <= MOST, "a tile ahead of the products");
};

// Two fp32 numbers at once (fma.rn.f32x2 and add.rn.f32x2: one issue slot for both).
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 f2(float a, float b) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void f2_get(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
// the larger of three, NaN if one is
__device__ __forceinline__ float max3_nan(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// 2^a, 2^b without the special-function unit: x = n + f with n the nearest whole number (added to 1.5 2^23 it stands in the last bits of the sum), 2^f on
// [-1/2, 1/2] by the cubic of least relative error among those with p(0) = 1 (1.0e-4; what it stands in for is rounded by up to 2^-8), n added to the exponent.  From
// -127 down the result is 0 (p = 1 there, and its exponent 127); a, b below 2^22 and not NaN.
__device__ __forceinline__ void exp2_pair(F2 x, float& a, float& b) {
  f2_get(x, a, b);
  x = f2(fmaxf(a, -127.0f), fmaxf(b, -127.0f));
  const F2 t = f2_add(x, f2(12582912.0f, 12582912.0f));
  const F2 n = f2_add(t, f2(-12582912.0f, -12582912.0f));
  const F2 f = f2_fma(n, f2(-1.0f, -1.0f), x);
  F2 p = f2_fma(f, f2(0.05500906f, 0.05500906f), f2(0.24221097f, 0.24221097f));
  p = f2_fma(p, f, f2(0.6932829f, 0.6932829f));
  p = f2_fma(p, f, f2(1.0f, 1.0f));
  float ta, tb;
  f2_get(t, ta, tb);
  f2_get(p, a, b);
  a = __int_as_float(__float_as_int(a) + (__float_as_int(ta) << 23));
  b = __int_as_float(__float_as_int(b) + (__float_as_int(tb) << 23));
}
constexpr int PX_POLY = 4;          // of 16 pairs of exponentials, how many run on the FMA units

struct PxParams {
  const __nv_bfloat16* q; int ldq;  // token t, head h at q + t · ldq + h · HD
  const float* cos_t; const float* sin_t; int max_pos; const int* cache_len;     // ROTATE: tables and the slot of the new token
  const int* prefix_len; const int* prefix_pad; const int* pad_left;
  __nv_bfloat16* out;
  float* o_part; float2* ml_part;   // partial triples [tokens · nh][parts]
  int S, rows, nh, nkv, gs, P, T, start;      // gs: log2 of the query heads per key head
  int shared, own, partial;         // which keys this launch visits; whether it leaves partial triples or the result
  int splits, parts, part0;         // splits of the shared keys in this launch; triples per (token, head), the first that this launch writes
  // the last `own_ctas` CTAs of a step, or a launch of their own, take the own keys, `own_splits` parts of every (token, key head)
  const __nv_bfloat16* prefix_k; const __nv_bfloat16* prefix_v; __nv_bfloat16* k_cache; __nv_bfloat16* v_cache;
  int own_ctas, own_splits, B, tiles_q;
  int p_low;                        // a step, or one tile of queries: probabilities as two bfloat16 numbers
  float scale_log2;
};

__device__ __forceinline__ void px_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void px_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void px_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// The own keys of a step (ROTATE), or of prompts of a few tokens, whose tiles would be all but empty.  A warp takes units, a part of the keys of one (token, key head), one after the other; its ring holds the next blocks of the same or the
// following unit.  As in decode_attn_fused.cu the G query heads are rows 0..G-1 of mma.sync operands of 16 rows, which leaves rows 8..15 for the low parts
// of the queries (scores) and of the probabilities (values): both keep 16 bits at no cost.  The new token of a step's row, in the last part, is folded in from
// registers; a prompt's tokens are in the cache.  Bound by the cache's bytes; a block's chain of dependent steps takes about 0.6 us, so that a warp moves 13 GB/s and eight of them an SM's share
// of the bandwidth twice over.
// KIND: what the units are.
constexpr int PX_PROMPT_OWN = 0, PX_STEP_OWN = 1, PX_STEP_ALL = 2;    // ALL: parts of the shared keys too, for the up to eight queries of a (group, key head)
template <int HD, int KIND>
__device__ __forceinline__ void px_own_keys(const PxParams& p, uint8_t* smem) {
  using Own = PxOwn<HD>;
  constexpr bool ROTATE = KIND != PX_PROMPT_OWN, ALL = KIND == PX_STEP_ALL;
  constexpr int KPI = Own::KPI, HALVES = Own::HALVES, STAGES = Own::STAGES;
  constexpr int NT = KPI / 8, NB = KPI / 16, KS = HD / 16;
  constexpr int CH = HD / 8, RPS = 32 / CH, PASSES = 8 / RPS;       // 16-byte chunks of a row, rows that a warp holds at once
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (warp >= Own::WARPS) return;
  const uint32_t raw = tc::smem_u32(smem), base0 = (raw + 1023u) & ~1023u;
  const uint32_t ring = base0 + warp * Own::RING, qt = base0 + Own::WARPS * Own::RING + warp * Own::QT;
  for (int i = lane; i < (int)Own::QT / 16; i += 32)                  // rows without a head: zero, or what a unit before had there
    asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(qt + 16 * i), "r"(0) : "memory");
  __syncwarp();
  if constexpr (ROTATE) pdl_wait();
  pdl_launch_dependents();

  const int G = 1 << p.gs, shared_units = ALL ? p.B / p.rows * p.nkv * p.splits : 0;
  const int units = shared_units + p.B * p.S * p.nkv * p.own_splits, step = p.own_ctas * Own::WARPS;
  const int len = ROTATE ? min(max(*p.cache_len, 0), p.T) : 0;           // a step: keys in front of the new token
  auto shared_range = [&](int group, int& lo, int& hi) {
    lo = p.prefix_pad ? max(p.prefix_pad[group], 0) : 0;
    hi = max(p.prefix_len ? min(p.prefix_len[group], p.P) : p.P, lo);
  };
  // first and last + 1 key of unit u, and its (row or group, key head) in the caches
  auto range = [&](int u, int& lo, int& hi, int& at) {
    int parts = p.own_splits, part, n;
    if (ALL && u < shared_units) {
      parts = p.splits;
      at = u / parts; part = u - at * parts;
      shared_range(at / p.nkv, lo, hi);
      n = hi - lo;
    } else {
      if (ALL) u -= shared_units;
      const int item = u / parts, token = item / p.nkv, b = ROTATE ? token : token / p.S;
      part = u - item * parts;
      at = ROTATE ? item : b * p.nkv + item - token * p.nkv;
      lo = p.pad_left ? max(p.pad_left[b], 0) : 0;
      n = max((ROTATE ? len : p.start + token - b * p.S + 1) - lo, 0);
    }
    const int chunk = ((n + parts - 1) / parts + KPI - 1) / KPI * KPI;
    hi = lo + min((part + 1) * chunk, n);
    lo += min(part * chunk, n);
  };
  // what is asked for next: block [r_base, r_base + KPI) of unit r_u
  const int first_unit = ((int)blockIdx.x - ((int)gridDim.x - p.own_ctas)) * Own::WARPS + warp;
  int r_u = first_unit, r_base = 0, r_hi = 0, r_at = 0, r_st = 0;
  if (r_u < units) range(r_u, r_base, r_hi, r_at);
  // 16-byte copies into the swizzled layout, eight 512-byte rows of requests each for keys and values; keys behind the last one become zeros (a weight of
  // zero times a NaN is a NaN).  By TMA, whose boxes of 16 rows leave the SM at 28 bytes a cycle, the warps waited for its queue a third of their time.
  const int r_ch = lane % CH, r_key = lane / CH;
  auto request = [&]() {
    while (r_u < units && r_base >= r_hi) {
      r_u += step;
      if (r_u < units) range(r_u, r_base, r_hi, r_at);
    }
    if (r_u < units) {
      const bool sh = ALL && r_u < shared_units;
      const __nv_bfloat16* from_k = sh ? p.prefix_k : p.k_cache;
      const __nv_bfloat16* from_v = sh ? p.prefix_v : p.v_cache;
      const uint32_t dst = ring + r_st * Own::STAGE + (r_ch >> 3) * Own::BOX;
      const size_t src = ((size_t)r_at * (sh ? p.P : p.T) + r_base + r_key) * HD + 8 * r_ch;
#pragma unroll
      for (int i = 0; i < KPI / RPS; ++i) {
        const int key = i * RPS + r_key;
        const uint32_t at = dst + key * 128 + (((r_ch & 7) ^ (key & 7)) << 4);
        const bool on = r_base + key < r_hi;
        const size_t from = on ? src + (size_t)(i * RPS) * HD : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from_k + from), "r"(on ? 16 : 0) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + HALVES * Own::BOX), "l"(from_v + from), "r"(on ? 16 : 0) : "memory");
      }
      r_base += KPI;
      if (++r_st == STAGES) r_st = 0;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");       // (a group per block or an empty one: the count of groups behind a block stays the same)
  };
#pragma unroll
  for (int i = 0; i < STAGES; ++i) request();

  // ldmatrix addresses within a 64-column box: row r's 16-byte chunk c lies at r * 128 + ((c ^ (r & 7)) << 4)
  const int l7 = lane & 7, q8 = lane >> 3;
  uint32_t koff[2], voff[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) koff[i] = l7 * 128 + (((4 * i + q8) ^ l7) << 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) voff[i] = ((q8 & 1) * 8 + l7) * 128 + (((2 * i + (q8 >> 1)) ^ l7) << 4);

  int st = 0;
#pragma unroll 1
  for (int u = first_unit; u < units; u += step) {
    int lo, hi, at_row;
    range(u, lo, hi, at_row);
    // queries of the unit: n of them, number r of token b + r / G and head r % G of the key head
    const bool sh = ALL && u < shared_units;
    const int parts = sh ? p.splits : p.own_splits, own_u = sh ? u : u - shared_units, item = own_u / parts, part = own_u - item * parts;
    const int kvh = item % p.nkv, b = sh ? item / p.nkv * p.rows : item / p.nkv, n = sh ? p.rows * G : G;
    auto row_of = [&](int r) { return p.q + (size_t)(b + (r >> p.gs)) * p.ldq + (size_t)(kvh * G + (r & (G - 1))) * HD; };
    const bool newest = ROTATE && !sh && part == p.own_splits - 1;
    // ---- queries: chunk `ch` of rows pass · RPS + lane / CH; and of the new token's key and value
    const int ch = lane % CH, rr = lane / CH;
    uint4 qx[PASSES], kx = make_uint4(0, 0, 0, 0), vx = kx;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
      if (i * RPS + rr < n) qx[i] = *reinterpret_cast<const uint4*>(row_of(i * RPS + rr) + 8 * ch);
    constexpr int NP = ALL ? PASSES : 1;         // rows of several tokens have angles of their own
    float cs[NP][4], sn[NP][4];
    if constexpr (ROTATE) {
      if (newest) {
        const __nv_bfloat16* row = p.q + (size_t)b * p.ldq;
        kx = *reinterpret_cast<const uint4*>(row + (size_t)(p.nh + kvh) * HD + 8 * ch);
        vx = *reinterpret_cast<const uint4*>(row + (size_t)(p.nh + p.nkv + kvh) * HD + 8 * ch);
      }
      int g_lo, g_hi;
      shared_range(b / p.rows, g_lo, g_hi);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int token = ALL ? b + (min(i * RPS + rr, n - 1) >> p.gs) : b;
        int pos = g_hi - g_lo + len - (p.pad_left ? p.pad_left[token] : 0);
        pos = pos < 0 ? 0 : (pos >= p.max_pos ? p.max_pos - 1 : pos);
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos_t) + (size_t)pos * CH + ch);
        const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin_t) + (size_t)pos * CH + ch);
        cs[i][0] = c4.x; cs[i][1] = c4.y; cs[i][2] = c4.z; cs[i][3] = c4.w;
        sn[i][0] = s4.x; sn[i][1] = s4.y; sn[i][2] = s4.z; sn[i][3] = s4.w;
      }
    }
    float kf[8];                                 // the new key, rotated and rounded as the cache holds it
    if constexpr (ROTATE) {
      const uint32_t x[4] = {kx.x, kx.y, kx.z, kx.w};
      uint32_t a[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float re = bf16_lo(x[e]), im = bf16_hi(x[e]);
        a[e] = pack_bf16(re * cs[0][e] - im * sn[0][e], re * sn[0][e] + im * cs[0][e]);
        kf[2 * e] = bf16_lo(a[e]); kf[2 * e + 1] = bf16_hi(a[e]);
      }
      if (newest && rr == 0 && len < p.T) {
        const size_t slot = ((size_t)at_row * p.T + len) * HD + 8 * ch;
        *reinterpret_cast<uint4*>(p.k_cache + slot) = make_uint4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<uint4*>(p.v_cache + slot) = vx;
      }
    }
    float s_new = 0.f;                           // of row g
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      if (i * RPS >= n) continue;                // warp-uniform
      const int r = i * RPS + rr;
      float dot = 0.f;
      if (r < n) {
        const uint32_t at = qt + r * (HD * 2) + ((ch ^ r) << 4);
        if constexpr (ROTATE) {
          const uint32_t x[4] = {qx[i].x, qx[i].y, qx[i].z, qx[i].w};
          uint32_t a[4], c[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float re = bf16_lo(x[e]), im = bf16_hi(x[e]);
            const float y = re * cs[i % NP][e] - im * sn[i % NP][e], z = re * sn[i % NP][e] + im * cs[i % NP][e];
            a[e] = pack_bf16(y, z);
            c[e] = pack_bf16(y - bf16_lo(a[e]), z - bf16_hi(a[e]));
            dot = fmaf(y, kf[2 * e], fmaf(z, kf[2 * e + 1], dot));
          }
          qx[i] = make_uint4(a[0], a[1], a[2], a[3]);
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + 8 * HD * 2), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]) : "memory");
        }
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(qx[i].x), "r"(qx[i].y), "r"(qx[i].z), "r"(qx[i].w) : "memory");
      }
      if (newest) {
#pragma unroll
        for (int d = CH / 2; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        const float mine = __shfl_sync(0xffffffffu, dot, (g % RPS) * CH);
        if (g / RPS == i) s_new = mine;
      }
    }
    __syncwarp();
    uint32_t qa[KS][4];                          // k-steps of the 16 rows
#pragma unroll
    for (int s = 0; s < KS; ++s) px_ldsm(qt + ((q8 & 1) * 8 + l7) * (HD * 2) + (((2 * s + (q8 >> 1)) ^ l7) << 4), qa[s]);
    if (newest) {                                // the new values wait where the queries were
      __syncwarp();
      if (rr == 0) asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(qt + 16 * ch), "r"(vx.x), "r"(vx.y), "r"(vx.z), "r"(vx.w) : "memory");
      __syncwarp();
    }

    float m = -INFINITY, l = 0.f;                // row g: m is quad-uniform, l is this thread's share of the sum
    float o[HD / 8][4];                          // [0..1]: row g against P's high parts, [2..3]: against the low parts
#pragma unroll
    for (int e = 0; e < HD / 8; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[e][i] = 0.f;
#pragma unroll 1
    for (int base = lo; base < hi; base += KPI) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const uint32_t ks = ring + st * Own::STAGE, vs = ks + HALVES * Own::BOX;
      // operands ahead of the products that take them: a load in front of each is 30 cycles apiece
      uint32_t kr[NT][KS / 2][4];
#pragma unroll
      for (int i = 0; i < KS / 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) px_ldsm(ks + (i >> 1) * Own::BOX + j * 1024 + koff[i & 1], kr[j][i]);
      float d[NT][2][4] = {};                    // two chains per 8 keys: half the latency of the dependent products
#pragma unroll
      for (int i = 0; i < KS / 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          px_mma(d[j][0], qa[2 * i][0], qa[2 * i][1], qa[2 * i][2], qa[2 * i][3], kr[j][i][0], kr[j][i][1]);
          px_mma(d[j][1], qa[2 * i + 1][0], qa[2 * i + 1][1], qa[2 * i + 1][2], qa[2 * i + 1][3], kr[j][i][2], kr[j][i][3]);
        }
      uint32_t vr[NB][HD / 16][4];
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int e = 0; e < HD / 16; ++e) px_ldsm_t(vs + (e >> 2) * Own::BOX + kb * 2048 + voff[e & 3], vr[kb][e]);
      __syncwarp();                              // every lane has read the stage: it may be filled again
      request();
      if (++st == STAGES) st = 0;
      float c[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int key = base + 8 * j + 2 * t;
        c[j][0] = key < hi ? ((d[j][0][0] + d[j][1][0]) + (d[j][0][2] + d[j][1][2])) * p.scale_log2 : -INFINITY;
        c[j][1] = key + 1 < hi ? ((d[j][0][1] + d[j][1][1]) + (d[j][0][3] + d[j][1][3])) * p.scale_log2 : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < NT; ++j) mx = fmaxf(mx, fmaxf(c[j][0], c[j][1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m, mx), m_safe = m_new == -INFINITY ? 0.f : m_new;
      const float corr = exp2f(m - m_safe);
      m = m_new;
      float psum = 0.f;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        c[j][0] = exp2f(c[j][0] - m_safe);
        c[j][1] = exp2f(c[j][1] - m_safe);
        psum += c[j][0] + c[j][1];
      }
      l = l * corr + psum;
      if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
        for (int e = 0; e < HD / 8; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[e][i] *= corr;
      }
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        const float(&c0)[2] = c[2 * kb];
        const float(&c1)[2] = c[2 * kb + 1];
        const uint32_t h0 = pack_bf16(c0[0], c0[1]), h2 = pack_bf16(c1[0], c1[1]);
        const uint32_t l0 = pack_bf16(c0[0] - bf16_lo(h0), c0[1] - bf16_hi(h0));
        const uint32_t l2 = pack_bf16(c1[0] - bf16_lo(h2), c1[1] - bf16_hi(h2));
#pragma unroll
        for (int e = 0; e < HD / 16; ++e) {
          px_mma(o[2 * e], h0, l0, h2, l2, vr[kb][e][0], vr[kb][e][1]);
          px_mma(o[2 * e + 1], h0, l0, h2, l2, vr[kb][e][2], vr[kb][e][3]);
        }
      }
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int row = g < n ? g : 0;
    const size_t th = (size_t)(b + (row >> p.gs)) * p.nh + kvh * G + (row & (G - 1)), at = th * p.parts + (sh ? 0 : p.splits) + part;
    float w_old = 1.f, w_new = 0.f;
    if (newest) {                                // one more key
      s_new *= p.scale_log2;
      const float m_new = fmaxf(m, s_new), m_safe = m_new == -INFINITY ? 0.f : m_new;
      w_old = exp2f(m - m_safe);
      w_new = exp2f(s_new - m_safe);
      l = l * w_old + w_new;
      m = m_new;
    }
    float* dst = p.o_part + at * HD;
#pragma unroll
    for (int e = 0; e < HD / 8; ++e) {
      float x = o[e][0] + o[e][2], y = o[e][1] + o[e][3];
      if (newest) {
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(qt + 16 * e + 4 * t) : "memory");
        x = fmaf(w_new, bf16_lo(v), x * w_old);
        y = fmaf(w_new, bf16_hi(v), y * w_old);
      }
      if (g < n && l != 0.f) *reinterpret_cast<float2*>(dst + 8 * e + 2 * t) = make_float2(x, y);
    }
    if (g < n && t == 0) p.ml_part[at] = make_float2(m, l);
    __syncwarp();                                // the next unit's queries take the place of the new values
  }
}

// The own keys of prompts of a few tokens, behind the launch over the shared ones.  It starts on SMs that this one leaves: every CTA there has waited for what ran
// before it lets a launch behind it begin, so nothing that is read here is still being written, and the wait is at the end, for the launch that joins both.
template <int HD>
__global__ void __launch_bounds__(256, 1) prefix_own_kernel(const PxParams p) {
  extern __shared__ __align__(1024) uint8_t px_smem[];
  px_own_keys<HD, PX_PROMPT_OWN>(p, px_smem);
  pdl_wait();
}

// A step whose groups have up to eight queries of a key head: both sets of keys by warps.
template <int HD>
__global__ void __launch_bounds__(256, 1) prefix_rows_kernel(const PxParams p) {
  extern __shared__ __align__(1024) uint8_t px_smem[];
  px_own_keys<HD, PX_STEP_ALL>(p, px_smem);
}

template <int HD, bool ROTATE, int MODE>
__global__ void __launch_bounds__(PxTile<HD, ROTATE, MODE>::THREADS, MODE == PX_SOLO ? 2 : 1)
prefix_attn_kernel(const __grid_constant__ CUtensorMap tm_pk, const __grid_constant__ CUtensorMap tm_pv,
                   const __grid_constant__ CUtensorMap tm_ok, const __grid_constant__ CUtensorMap tm_ov, const PxParams p) {
  using Tile = PxTile<HD, ROTATE, MODE>;
  constexpr bool PAIR = Tile::PAIR, SOLO = Tile::SOLO, JOINT = Tile::JOINT, LOW = !JOINT || ROTATE;      // LOW: probabilities may have low parts
  constexpr int HALVES = Tile::HALVES, NQ = Tile::NQ, SLOTS = Tile::SLOTS;
  extern __shared__ __align__(1024) uint8_t px_smem[];
  const uint32_t raw = tc::smem_u32(px_smem);
  const uint32_t base = (raw + 1023u) & ~1023u;  // the 128-byte swizzle counts rows from 1024-byte boundaries
  const uint32_t sQ = base, ring = base + Tile::QS, small = ring + SLOTS * Tile::SLOT;
  const uint32_t q_full = small, tmem_slot = small + 8;
  auto p_full = [&](int w, int i) { return small + 16 + 16u * w + 8u * (i & 1); };       // probabilities of a tile
  auto o_last = [&](int w, int i) { return small + 80 + 16u * w + 8u * (i & 1); };       // the last product but one, the last (one phase each)
  const uint32_t started = small + 120;                                // PAIR: the first set is through its first softmax
  auto s_full = [&](int w, int i) { return small + 48 + 16u * w + 8u * (i & 1); };       // scores of a tile
  auto slot_full = [&](int s) { return small + 128 + 16u * s; };
  auto slot_empty = [&](int s) { return small + 136 + 16u * s; };
  static_assert(128 + 16 * SLOTS <= 512, "barriers in front of the rows' statistics");
  float2* s_ml = reinterpret_cast<float2*>(px_smem + (small + 512 - raw));       // [2][128]
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(px_smem + (tmem_slot - raw));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = 1 << p.gs;
  if constexpr (ROTATE) {
    if ((int)blockIdx.x >= (int)gridDim.x - p.own_ctas) {
      px_own_keys<HD, PX_STEP_OWN>(p, px_smem);
      return;
    }
  }
  // z: group (shared keys alone) or row; kvh: key head; qt: query tile (or pair), longest first; split of the shared keys
  int idx = (int)blockIdx.x;
  const int split = idx % p.splits;
  idx /= p.splits;
  const int qt = p.tiles_q - 1 - idx % p.tiles_q;
  idx /= p.tiles_q;
  const int kvh = idx % p.nkv, z = idx / p.nkv;
  const int unit_tokens = p.own ? p.S : p.rows * p.S;             // tokens whose queries this launch packs together
  const int token0 = z * unit_tokens;
  const int q0 = qt * Tile::ROWS, n_rows = min(Tile::ROWS, unit_tokens * G - q0);
  const int group = p.own ? z / p.rows : z;
  const bool two = !SOLO && (!PAIR || n_rows > PX_BM);                       // the second set of softmax warps has work

  if (warp == 0 && lane == 0) {
    if (p.shared) { tc::prefetch_tensormap(&tm_pk); tc::prefetch_tensormap(&tm_pv); }
    if (p.own) { tc::prefetch_tensormap(&tm_ok); tc::prefetch_tensormap(&tm_ov); }
  }
  if (warp == 1 && lane == 0) {
    tc::mbar_init(q_full, 4 * Tile::SETS);
    tc::mbar_init(started, 1);
    const int users = JOINT && two ? 2 : 1;                        // products that read a tile
    for (int w = 0; w < 2; ++w) {
      tc::mbar_init(p_full(w, 0), 4); tc::mbar_init(p_full(w, 1), 4); tc::mbar_init(o_last(w, 0), 1); tc::mbar_init(o_last(w, 1), 1);
      tc::mbar_init(s_full(w, 0), 1); tc::mbar_init(s_full(w, 1), 1);
    }
    for (int s = 0; s < SLOTS; ++s) { tc::mbar_init(slot_full(s), 1); tc::mbar_init(slot_empty(s), users); }
    tc::fence_barrier_init();
  }
  if (warp == 0) tc::tmem_alloc(tmem_slot, 256 * Tile::SETS);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot_ptr;
  auto tS = [&](int w, int i) { return tmem + (uint32_t)w * 256u + (uint32_t)(i & 1) * 64u; };   // scores of tile i of set w, afterwards its probabilities
  auto tO = [&](int w) { return tmem + (uint32_t)w * 256u + 128u; };

  pdl_wait();
  pdl_launch_dependents();

  // shared keys [s_lo, s_hi) of this CTA, own keys [o_lo, o_hi)
  int s_lo = 0, s_hi = 0, o_lo = 0, o_hi = 0;
  const int g_lo = p.prefix_pad ? max(p.prefix_pad[group], 0) : 0;
  const int g_hi = p.prefix_len ? min(p.prefix_len[group], p.P) : p.P;
  const int pad = p.own && p.pad_left ? max(p.pad_left[z], 0) : 0;
  {
    const int n_sh = p.shared ? max(g_hi - g_lo, 0) : 0, sh_tiles = (n_sh + PX_BN - 1) / PX_BN;
    const int own_end = p.own ? max(p.start + ((q0 + n_rows - 1) >> p.gs) + 1, pad) : pad;       // slot of the tile's last token: its last key
    // this split's tiles [j0, j1) of the shared keys' and then the own keys'
    const int all = sh_tiles + (own_end - pad + PX_BN - 1) / PX_BN, per = (all + p.splits - 1) / p.splits;
    const int j0 = min(split * per, all), j1 = min(j0 + per, all);
    s_lo = g_lo + min(min(j0, sh_tiles) * PX_BN, n_sh);
    s_hi = g_lo + min(min(j1, sh_tiles) * PX_BN, n_sh);
    o_lo = min(pad + max(j0 - sh_tiles, 0) * PX_BN, own_end);
    o_hi = min(pad + max(j1 - sh_tiles, 0) * PX_BN, own_end);
  }
  const int n_shared = (s_hi - s_lo + PX_BN - 1) / PX_BN, n_tiles = n_shared + (o_hi - o_lo + PX_BN - 1) / PX_BN;
  // set w's tile i is tile number i (PAIR) or 2 i + w of the keys
  auto tiles_of = [&](int w) { return PAIR ? (w == 0 || two ? n_tiles : 0) : (n_tiles + 1 - w) / 2; };
  auto tile_at = [&](int w, int i) { return PAIR ? i : 2 * i + w; };

  if (warp == 0) {
    if (lane == 0) {
      int sl = 0;
      uint32_t ph = 1;
      for (int idx = 0; idx < (JOINT ? 1 : 2) * n_tiles; ++idx) {       // tiles, or K_0, V_0, K_1, V_1, ...
        const int j = JOINT ? idx : idx >> 1;
        const bool mine = j >= n_shared;
        const int key0 = mine ? o_lo + (j - n_shared) * PX_BN : s_lo + j * PX_BN;
        const int head = (mine ? z : group) * p.nkv + kvh;
        const CUtensorMap* mk = mine ? &tm_ok : &tm_pk;
        const CUtensorMap* mv = mine ? &tm_ov : &tm_pv;
        tc::mbar_wait(slot_empty(sl), ph);
        tc::mbar_expect_tx(slot_full(sl), Tile::SLOT);
        const CUtensorMap* m0 = !JOINT && (idx & 1) ? mv : mk;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) tc::tma_load_3d(ring + sl * Tile::SLOT + h * Tile::KV_HALF, m0, slot_full(sl), 64 * h, key0, head, tc::EVICT_NORMAL);
        if constexpr (JOINT) {
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            tc::tma_load_3d(ring + sl * Tile::SLOT + Tile::KV + h * Tile::KV_HALF, mv, slot_full(sl), 64 * h, key0, head, tc::EVICT_NORMAL);
        }
        if (++sl == SLOTS) { sl = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1 || warp == 10) {
    // a warp per set issues its products: the whole warp walks the loop, one elected lane issues; descriptors are advanced by their address field
    // (flash_prefill.cu).  Two warps, so that neither set waits for the other's softmax, and as few waits as there are tiles: a wait costs this warp some
    // 150 cycles even where nothing is left to wait for, and a loop with three of them and divisions took 1700 cycles per tile for 600 of products.
    const int w = warp == 1 ? 0 : 1, mine = tiles_of(w);
    constexpr uint32_t IDESC_S = tc::idesc_bf16_f32(PX_BM, PX_BN, false, false);
    constexpr uint32_t IDESC_O = tc::idesc_bf16_f32(PX_BM, HD, false, true);        // B = V is MN-major
    constexpr int STEP = JOINT ? 1 : 2 * Tile::SETS;                                 // slots from one of this set's tiles to the next
    const uint64_t dQ = tc::smem_desc_kmajor_sw128(sQ + (PAIR ? w * NQ * Tile::Q : 0));
    const uint64_t dK0 = tc::smem_desc_kmajor_sw128(ring);
    const uint64_t dV0 = tc::smem_desc_mnmajor_sw128(ring + (JOINT ? Tile::KV : 0), Tile::KV_HALF, 1024);
    int k_sl = JOINT ? 0 : 2 * w, v_sl = JOINT ? 0 : 2 * w + 1;          // slots of the next scores and of the next product
    uint32_t k_ph = 0, v_ph = 0;
    auto next_slot = [&](int& sl) { sl += STEP; if (sl >= SLOTS) { sl -= SLOTS; return 1u; } return 0u; };
    auto issue_s = [&](int i) {
      tc::mbar_wait(slot_full(k_sl), k_ph);
      tc::fence_after_sync();
      if (tc::elect_one()) {
        const uint64_t dK = dK0 + (uint64_t)k_sl * (Tile::SLOT >> 4);
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            tc::mma_ss(tS(w, i), dQ + (uint64_t)((n * Tile::Q + (k >> 2) * Tile::Q_HALF + (k & 3) * 32) >> 4),
                       dK + (uint64_t)(((k >> 2) * Tile::KV_HALF + (k & 3) * 32) >> 4), IDESC_S, n != 0 || k != 0);
        tc::mma_commit(s_full(w, i));
        if (!JOINT) tc::mma_commit(slot_empty(k_sl));
      }
      __syncwarp();
      k_ph ^= next_slot(k_sl);
    };
    if (mine > 0) {
      tc::mbar_wait(q_full, 0);
      tc::fence_after_sync();
      // the sets run half a tile apart, so that one's exponentials fall into the other's loads and waits; started together they stay together
      if (JOINT && w == 1) tc::mbar_wait(started, 0);
      issue_s(0);
    }
    for (int i = 0; i < mine; ++i) {
      if (i + 1 < mine) issue_s(i + 1);                                // the tensor core forms the next scores during this tile's softmax
      if (!JOINT) tc::mbar_wait(slot_full(v_sl), v_ph);
      const int j = tile_at(w, i);
      const int left = j < n_shared ? s_hi - s_lo - j * PX_BN : o_hi - o_lo - (j - n_shared) * PX_BN;
      if (left < PX_BN) {                                              // value rows that hold no key (both sets write the same zeros)
        for (int e = lane; e < (PX_BN - left) * 8 * HALVES; e += 32) {
          const int r = left + e / (8 * HALVES), c = e % (8 * HALVES);
          const uint32_t a = ring + v_sl * Tile::SLOT + (JOINT ? Tile::KV : 0) + (c >> 3) * Tile::KV_HALF + r * 128 + (c & 7) * 16;
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      tc::mbar_wait(p_full(w, i), (i >> 1) & 1);
      tc::fence_after_sync();
      if (tc::elect_one()) {
        const uint64_t dV = dV0 + (uint64_t)v_sl * (Tile::SLOT >> 4);
#pragma unroll
        for (int k = 0; k < (LOW ? 2 : 1) * PX_BN / 16; ++k)          // A = P in TMEM: 16 keys = 8 columns of packed pairs; the low parts behind the high ones
          if (k < 4 || p.p_low) tc::mma_ts(tO(w), tS(w, i) + k * 8, dV + (uint64_t)(((k & 3) * 2048) >> 4), IDESC_O, i != 0 || k != 0);
        tc::mma_commit(slot_empty(v_sl));
        if (i + 2 >= mine) tc::mma_commit(o_last(w, i + 2 - mine));
      }
      __syncwarp();
      v_ph ^= next_slot(v_sl);
    }
  } else {
    const int w = !SOLO && warp >= 6 ? 1 : 0;                                   // set of softmax warps (2..5, 6..9)
    const int quarter = warp & 3;                                      // TMEM lane quadrant of this warp
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    // ---- queries, 16 bytes per lane and step: a set's own tile, or half of the one tile
    constexpr int CH = HD / 8, RPS = 32 / CH;                          // 16-byte chunks of a row, rows of a step
    const int ch = lane % CH;
    if (n_tiles > 0) {
      constexpr int STEPS = (PAIR ? 32 : 16) / RPS, AHEAD = ROTATE ? 4 : 16;           // loads in flight
      const int row0 = (PAIR ? quarter * 32 : (w * 4 + quarter) * 16) + lane / CH;       // (rows behind the last query: zeros; their scores have a say in the way that a warp takes)
#pragma unroll 1
      for (int i0 = 0; i0 < STEPS; i0 += AHEAD) {
        uint4 x[AHEAD];
        float4 c4[ROTATE ? AHEAD : 1], s4[ROTATE ? AHEAD : 1];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int qr = (PAIR ? w * PX_BM : 0) + row0 + (i0 + u) * RPS;
          if (i0 + u < STEPS && qr < n_rows) {
            const int token = token0 + ((q0 + qr) >> p.gs), h = kvh * G + ((q0 + qr) & (G - 1));
            x[u] = *reinterpret_cast<const uint4*>(p.q + (size_t)token * p.ldq + (size_t)h * HD + 8 * ch);
            if constexpr (ROTATE) {
              int pos = max(g_hi - g_lo, 0) + min(max(*p.cache_len, 0), p.T) - (p.pad_left ? p.pad_left[token] : 0);
              pos = pos < 0 ? 0 : (pos >= p.max_pos ? p.max_pos - 1 : pos);
              c4[u] = __ldg(reinterpret_cast<const float4*>(p.cos_t) + (size_t)pos * CH + ch);
              s4[u] = __ldg(reinterpret_cast<const float4*>(p.sin_t) + (size_t)pos * CH + ch);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int r = row0 + (i0 + u) * RPS;
          if (i0 + u < STEPS) {
            const bool on = (PAIR ? w * PX_BM : 0) + r < n_rows;
            const uint32_t dst = sQ + (PAIR ? w * NQ * Tile::Q : 0) + (ch >> 3) * Tile::Q_HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
            if (!on) x[u] = make_uint4(0, 0, 0, 0);
            if constexpr (ROTATE) {
              const float cs[4] = {c4[u].x, c4[u].y, c4[u].z, c4[u].w}, sn[4] = {s4[u].x, s4[u].y, s4[u].z, s4[u].w};
              const uint32_t v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
              uint32_t a[4], b[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float re = bf16_lo(v[e]), im = bf16_hi(v[e]);
                const float y = re * cs[e] - im * sn[e], z_ = re * sn[e] + im * cs[e];
                a[e] = pack_bf16(y, z_);
                b[e] = pack_bf16(y - bf16_lo(a[e]), z_ - bf16_hi(a[e]));
              }
              if (on) x[u] = make_uint4(a[0], a[1], a[2], a[3]);
              else b[0] = b[1] = b[2] = b[3] = 0;
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + Tile::Q), "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3]) : "memory");
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(x[u].x), "r"(x[u].y), "r"(x[u].z), "r"(x[u].w) : "memory");
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full);
    }

    const int r = quarter * 32 + lane, qr = (PAIR ? w * PX_BM : 0) + r;               // this thread's query
    const int warp_row = (PAIR ? w * PX_BM : 0) + quarter * 32;                        // the warp's first
    const bool row_on = qr < n_rows, warp_on = warp_row < n_rows;
    const int at = q0 + min(qr, n_rows - 1);
    const int slot = p.own ? p.start + (at >> p.gs) : 0;                                     // of the query's own key
    const int slot_warp = p.own ? p.start + ((q0 + min(warp_row, n_rows - 1)) >> p.gs) : 0;  // the smallest of the warp
    const int my_tiles = tiles_of(w);
    float m_ref = -INFINITY, l_run = 0.f;
    for (int i = 0; i < my_tiles; ++i) {
      const int j = tile_at(w, i);
      const bool mine = j >= n_shared;
      const int key0 = mine ? o_lo + (j - n_shared) * PX_BN : s_lo + j * PX_BN;
      const int end = mine ? slot + 1 : s_hi;                          // first key that this row does not see
      const int end_warp = mine ? slot_warp + 1 : s_hi;                // the smallest of the warp
      tc::mbar_wait(s_full(w, i), (i >> 1) & 1);
      tc::fence_after_sync();
      if (warp_on) {
        uint32_t v0[32], v1[32];
        tc::tmem_ld32(tS(w, i) + lane_off, v0);
        tc::tmem_ld32(tS(w, i) + lane_off + 32, v1);
        tc::tmem_ld_wait();
        if (key0 + PX_BN > end_warp) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (key0 + e >= end) v0[e] = 0xff800000u;                  // -inf
            if (key0 + 32 + e >= end) v1[e] = 0xff800000u;
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; ++e) mx4[e & 3] = max3_nan(mx4[e & 3], __uint_as_float(v0[e]), __uint_as_float(v1[e]));
        const float t = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * p.scale_log2;
        const bool need = t > m_ref + PX_RESCALE || (m_ref == -INFINITY && t > -INFINITY);
        bool odd = !(t < INFINITY);                                    // NaN or infinite scores show in the result: no shortcuts
        if (i == 0) m_ref = t;
        if (__any_sync(0xffffffffu, odd || (i > 0 && need))) {
          odd = __any_sync(0xffffffffu, odd);
          if (i > 0 && __any_sync(0xffffffffu, need)) {
            const float factor = need ? exp2f(m_ref - t) : 1.0f;       // m_ref = -inf: 0 (O and l are 0 there)
            // O at rest: the next scores are issued behind product i - 1
            if (i + 1 < my_tiles) tc::mbar_wait(s_full(w, i + 1), ((i + 1) >> 1) & 1);
            else tc::mbar_wait(o_last(w, 0), 0);
            tc::fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tc::tmem_ld32(tO(w) + lane_off + c * 32, o);
              tc::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
              tc::tmem_st32(tO(w) + lane_off + c * 32, o);
            }
            tc::tmem_st_wait();
            l_run *= factor;
            if (need) m_ref = t;
          }
        }
        const float m_safe = m_ref == -INFINITY ? 0.f : m_ref;
        F2 sum = f2(0.f, 0.f);
        uint32_t hi[32], lo[LOW ? 32 : 1];
        const F2 scale2 = f2(p.scale_log2, p.scale_log2), minus_m = f2(-m_safe, -m_safe);
        auto pair = [&](int e, bool poly) {                            // keys 2e, 2e + 1
          const uint32_t* v = e < 16 ? v0 + 2 * e : v1 + 2 * e - 32;
          const F2 x = f2_fma(f2(__uint_as_float(v[0]), __uint_as_float(v[1])), scale2, minus_m);
          float a, b;
          if (poly) {
            exp2_pair(x, a, b);
          } else {
            f2_get(x, a, b);
            a = exp2f(a); b = exp2f(b);
          }
          sum = f2_add(sum, f2(a, b));
          hi[e] = pack_bf16(a, b);
          if (LOW && p.p_low) lo[LOW ? e : 0] = pack_bf16(a - bf16_lo(hi[e]), b - bf16_hi(hi[e]));
        };
        if (!odd && (!LOW || !p.p_low)) {
#pragma unroll
          for (int e = 0; e < 32; ++e) pair(e, (e * PX_POLY) % 16 < PX_POLY);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) pair(e, false);
        }
        float psum, psum2;
        f2_get(sum, psum, psum2);
        psum += psum2;
        tc::tmem_st32(tS(w, i) + lane_off, hi);                        // keys 2c, 2c + 1 of this row: 32-bit column c
        if constexpr (LOW) if (p.p_low) tc::tmem_st32(tS(w, i) + lane_off + 32, lo);
        tc::tmem_st_wait();
        l_run += psum;
      }
      // (two barriers in turn: this warp's next arrival at the same one comes after scores that the MMA warp forms behind its wait for this phase)
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_full(w, i));
      if (JOINT && i == 0 && warp == 2 && lane == 0) tc::mbar_arrive(started);
    }
    if (my_tiles > 0) {
      tc::mbar_wait(o_last(w, 1), 0);
      tc::fence_after_sync();
    }

    // ---- one triple per row: o = f0 O_0 + f1 O_1 against M.  Without PAIR both sets of warps hold the same rows: each takes half of the columns
    float M = l_run != 0.f ? m_ref : -INFINITY, L = l_run, f0 = l_run != 0.f ? 1.f : 0.f, f1 = 0.f;       // (a sum of zero: no keys; NaN stays NaN)
    if constexpr (!PAIR) {
      float2* other = s_ml + r + 128 * (1 - w);
      s_ml[r + 128 * w] = make_float2(m_ref, l_run);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (tiles_of(1 - w) > 0) {
        tc::mbar_wait(o_last(1 - w, 1), 0);
        tc::fence_after_sync();
      }
      const float2 o = *other;
      if (o.y != 0.f) M = fmaxf(M, o.x);
      const float Ms = M == -INFINITY ? 0.f : M;
      const float mine = l_run != 0.f ? exp2f(m_ref - Ms) : 0.f, theirs = o.y != 0.f ? exp2f(o.x - Ms) : 0.f;
      L = l_run * mine + o.y * theirs;
      f0 = w == 0 ? mine : theirs;
      f1 = w == 0 ? theirs : mine;
    }
    if (warp_on) {
      const int th = (token0 + (at >> p.gs)) * p.nh + kvh * G + (at & (G - 1));       // (token, head) of this row
      constexpr int CHUNKS = HD / 32 / (PAIR ? 1 : 2);
      // a row is a thread here and a run of memory there: 32 x 32 values change hands in shared memory that no product reads any more (the set's own queries, or the
      // ring when both sets are through), so that a store covers whole rows of 128 or 64 bytes
      const uint32_t stage = PAIR ? sQ + w * NQ * Tile::Q + quarter * 4096 : ring + (w * 4 + quarter) * 4096;
      const float inv = !p.partial && row_on && slot >= pad && L != 0.f ? 1.0f / L : 0.f;       // a query in front of its row's first token is padding: zeros
      const size_t part = (size_t)p.part0 + split;
      if (p.partial && row_on && (PAIR || w == 0)) p.ml_part[(size_t)th * p.parts + part] = make_float2(M, slot >= pad ? L : 0.f);
#pragma unroll 1
      for (int k = 0; k < CHUNKS; ++k) {
        const int c = (PAIR ? 0 : w * CHUNKS) + k;                     // columns [32 c, 32 c + 32)
        float o[32];
        {
          uint32_t a[32];
          if (__any_sync(0xffffffffu, f0 != 0.f)) {
            tc::tmem_ld32(tO(PAIR ? w : 0) + lane_off + c * 32, a);
            tc::tmem_ld_wait();
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = f0 != 0.f ? __uint_as_float(a[e]) * f0 : 0.f;
          if constexpr (!PAIR) {
            if (__any_sync(0xffffffffu, f1 != 0.f)) {
              tc::tmem_ld32(tO(1) + lane_off + c * 32, a);
              tc::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] += f1 != 0.f ? __uint_as_float(a[e]) * f1 : 0.f;
            }
          }
        }
        if (p.partial) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 128 + ((e ^ (lane & 7)) << 4)), "f"(o[4 * e]), "f"(o[4 * e + 1]), "f"(o[4 * e + 2]),
                         "f"(o[4 * e + 3]) : "memory");
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r2 = 4 * i + (lane >> 3), th2 = __shfl_sync(0xffffffffu, th, r2);
            float4 v;
            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(stage + r2 * 128 + (((lane ^ r2) & 7) << 4)) : "memory");
            if (warp_row + r2 < n_rows) *reinterpret_cast<float4*>(p.o_part + ((size_t)th2 * p.parts + part) * HD + 32 * c + 4 * (lane & 7)) = v;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            auto v = [&](int i) { return inv != 0.f ? o[8 * e + i] * inv : 0.f; };
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)), "r"(pack_bf16(v(0), v(1))),
                         "r"(pack_bf16(v(2), v(3))), "r"(pack_bf16(v(4), v(5))), "r"(pack_bf16(v(6), v(7))) : "memory");
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r2 = 8 * i + (lane >> 2), th2 = __shfl_sync(0xffffffffu, th, r2);
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(stage + r2 * 64 + (((lane ^ (r2 >> 1)) & 3) << 4)) : "memory");
            if (warp_row + r2 < n_rows) *reinterpret_cast<uint4*>(p.out + (size_t)th2 * HD + 32 * c + 8 * (lane & 3)) = v;
          }
        }
        __syncwarp();
      }
    }
    tc::fence_before_sync();
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, 256 * Tile::SETS);
}

// Joins the triples of a (token, head), a warp each.  `own`: the part of the own keys of a prompt, -1 where every part says itself that a query
// is padding: without own keys, or without any, it gives zeros.
template <int HD>
__global__ void __launch_bounds__(256) prefix_join_kernel(const float* __restrict__ o_part, const float2* __restrict__ ml_part, __nv_bfloat16* out, int rows, int parts, int own) {
  constexpr int V = HD / 32, AT_ONCE = 16;                             // columns of a lane, rows in flight
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  if (row >= rows) return;
  const float2* ml = ml_part + (size_t)row * parts;
  float m[3], w[3], M = -INFINITY, L = 0.f;                            // parts i, i + 32, i + 64
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float2 v = lane + 32 * k < parts ? __ldcg(ml + lane + 32 * k) : make_float2(-INFINITY, 0.f);
    m[k] = v.x; w[k] = v.y;
    if (w[k] != 0.f) M = fmaxf(M, m[k]);                               // (a sum of zero: no keys, and no o was written; NaN stays NaN)
  }
  M = warp_max(M);
  if (M == -INFINITY) M = 0.f;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float f = w[k] != 0.f ? exp2f(m[k] - M) : 0.f;
    L += f * w[k];
    w[k] = f;
  }
  L = warp_sum(L);
  const float* src = o_part + (size_t)row * parts * HD + V * lane;
  float acc[V] = {};
#pragma unroll 1
  for (int i0 = 0; i0 < parts; i0 += AT_ONCE) {                        // that many rows requested before the first is used
    float x[AT_ONCE][V], f[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int i = i0 + u, k = i >> 5;
      f[u] = __shfl_sync(0xffffffffu, k == 0 ? w[0] : (k == 1 ? w[1] : w[2]), i & 31);
      if (i >= parts) f[u] = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) x[u][e] = 0.f;
      if (f[u] != 0.f) {
        if constexpr (V == 4) {
          const float4 a = __ldcg(reinterpret_cast<const float4*>(src + (size_t)i * HD));
          x[u][0] = a.x; x[u][1] = a.y; x[u][2] = a.z; x[u][3] = a.w;
        } else {
          const float2 a = __ldcg(reinterpret_cast<const float2*>(src + (size_t)i * HD));
          x[u][0] = a.x; x[u][1] = a.y;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(f[u], x[u][e], acc[e]);
  }
  const bool seen = L != 0.f && (own < 0 || ml[own].y != 0.f);         // (the same address for the warp)
  const float inv = seen ? 1.f / L : 0.f;
  uint32_t* dst = reinterpret_cast<uint32_t*>(out + (size_t)row * HD + V * lane);
  if (!seen)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
  if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
  else *dst = pack_bf16(acc[0] * inv, acc[1] * inv);
}

// (attributes belong to the device's context: set at the first call on each, a bit per device; setting them twice is harmless)
static int px_smem_set(std::atomic<uint64_t>& set, const void* kernel, uint32_t smem) {
  int dev = 0;
  JL_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit == 0 || !(set.load(std::memory_order_acquire) & bit)) {
    JL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    set.fetch_or(bit, std::memory_order_release);
  }
  return JL_OK;
}

template <int HD, bool ROTATE, int MODE>
static int px_launch(const PxParams& p, unsigned ctas, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& ok, const CUtensorMap& ov, cudaStream_t st) {
  using Tile = PxTile<HD, ROTATE, MODE>;
  static std::atomic<uint64_t> set{0};
  const int rc = px_smem_set(set, (const void*)prefix_attn_kernel<HD, ROTATE, MODE>, Tile::SMEM);
  if (rc != JL_OK) return rc;
  JL_CUDA(launch_pdl(prefix_attn_kernel<HD, ROTATE, MODE>, dim3(ctas), dim3(Tile::THREADS), (size_t)Tile::SMEM, st, pk, pv, ok, ov, p));
  return JL_OK;
}

template <int HD, bool STEP>
static int px_warps_launch(const PxParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> set{0};
  void (*const kernel)(const PxParams) = STEP ? prefix_rows_kernel<HD> : prefix_own_kernel<HD>;
  const int rc = px_smem_set(set, (const void*)kernel, PxOwn<HD>::SMEM);
  if (rc != JL_OK) return rc;
  JL_CUDA(launch_pdl(kernel, dim3((unsigned)p.own_ctas), dim3(256), (size_t)PxOwn<HD>::SMEM, st, p));
  return JL_OK;
}

static int px_join(const PxParams& p, __nv_bfloat16* out, int rows, int hd, int own, cudaStream_t st) {
  const dim3 grid((unsigned)((rows + 7) / 8));
  if (hd == 128) JL_CUDA(launch_pdl(prefix_join_kernel<128>, grid, dim3(256), 0, st, (const float*)p.o_part, (const float2*)p.ml_part, out, rows, p.parts, own));
  else JL_CUDA(launch_pdl(prefix_join_kernel<64>, grid, dim3(256), 0, st, (const float*)p.o_part, (const float2*)p.ml_part, out, rows, p.parts, own));
  return JL_OK;
}

constexpr int PX_MAX_SPLITS = 64, PX_MAX_OWN = 16, PX_SMS = 148;

static long px_tiles(long queries) { return queries > PX_BM ? (queries + 2 * PX_BM - 1) / (2 * PX_BM) : 1; }

// One launch over tiles of the queries of `units` groups or rows, `queries` of a key head each.
static int px_dispatch(PxParams p, long queries, int units, bool rotate, int hd, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& ok,
                       const CUtensorMap& ov, cudaStream_t st) {
  // Two CTAs to an SM where tiles outnumber the SMs, and for larger prompts over few keys, where what a CTA does beside its tiles counts most: us in a graph, pairs and
  // this, 26 x 146 tokens x 32 key heads over 35 keys 76, 59; 10 x 403 over 47 54, 46; 8 x 64 x 4 over 500 (64 pairs) 14.8, 12.2, over 1000 22, 18; 16 x 128 x 4 over 100 21.6, 20.4; and over
  // 1000 44, 47, 4000 120, 135: every CTA then asks L2 for keys of its own.
  const float keys = (p.shared ? (float)p.P : 0.f) + (p.own ? (float)p.start + 0.5f * (float)p.S : 0.f), tiles = keys / (float)(PX_BN * p.splits);
  const long pairs = px_tiles(queries) * p.splits * p.nkv * units;
  const bool solo = !rotate && (queries <= PX_BM ? pairs > PX_SMS : tiles <= (2 * pairs <= PX_SMS ? 20.f : 8.f));
  const int mode = solo ? PX_SOLO : (queries > PX_BM ? PX_PAIR : PX_TURNS);
  p.tiles_q = solo ? (int)((queries + PX_BM - 1) / PX_BM) : (int)px_tiles(queries);
  p.p_low = rotate || queries <= PX_BM;
  const long ctas = p.own_ctas + (long)p.tiles_q * p.splits * p.nkv * units;
  JL_CHECK_ARG(ctas < (1l << 31), "attention over a shared prefix: %ld tiles", ctas);
#define JL_PX(HD_, R_, M_) if (hd == HD_ && rotate == R_ && mode == M_) return px_launch<HD_, R_, M_>(p, (unsigned)ctas, pk, pv, ok, ov, st);
  JL_PX(128, true, PX_PAIR) JL_PX(128, true, PX_TURNS) JL_PX(128, false, PX_PAIR) JL_PX(128, false, PX_TURNS) JL_PX(128, false, PX_SOLO)
  JL_PX(64, true, PX_PAIR) JL_PX(64, true, PX_TURNS) JL_PX(64, false, PX_PAIR) JL_PX(64, false, PX_TURNS) JL_PX(64, false, PX_SOLO)
#undef JL_PX
  return JL_ERR_UNSUPPORTED;
}


// Time of a launch in units of a tile of keys: rounds of CTAs (one per SM; `solo`: two where one tile of queries has more of them) times the tiles of one and its
// way in and out.
static float px_rounds(long queries, long units, int nkv, int splits, float tiles, bool solo) {
  const long full = queries > PX_BM ? queries / (2 * PX_BM) : 1, rest = px_tiles(queries) - full;      // whole pairs, one that may be half a pair
  const long ctas = (full + rest) * units * nkv * splits;
  if (solo && queries <= PX_BM && ctas > PX_SMS) return (float)((ctas + 2 * PX_SMS - 1) / (2 * PX_SMS)) * (1.35f * tiles + 8.f);
  const float whole = tiles + 5.f, part = rest && queries % (2 * PX_BM) <= PX_BM ? 0.78f * tiles + 5.f : whole;
  if (part == whole || ctas <= PX_SMS) return (float)((ctas + PX_SMS - 1) / PX_SMS) * (full ? whole : part);
  return (float)(units * nkv * splits) * (full * whole + rest * part) / PX_SMS + 0.5f * whole;
}

// Splits of the shared keys: the count with the least time, every one two tiles of keys or more; a split costs the triples' way to memory and back.
static int px_splits(long queries, int groups, int nkv, int prefix, bool solo = false, float* cost = nullptr) {
  const int tiles = (prefix + PX_BN - 1) / PX_BN;
  int best = 1;
  float least = 0.f;
  for (int s = 1; s <= PX_MAX_SPLITS && (s == 1 || 2 * s <= tiles); ++s) {
    const float c = px_rounds(queries, groups, nkv, s, (float)((tiles + s - 1) / s), solo) + (float)(queries * groups * nkv) * s * 3e-4f;
    if (s == 1 || c < least) { least = c; best = s; }
  }
  if (cost) *cost = least;
  return best;
}

// A step: CTAs and parts for the own keys, splits for the shared keys.  The shared keys' CTAs come first in the grid and the own keys', a unit for every warp, take the
// SMs that are left and those that get free: how full the caches are is known on the device alone, and an order that is right at any fill beats a division of the
// SMs between the two (us on one B200, a division by estimate, the best of all divisions, this: 96 rows over 32768 shared, with probabilities of one number, 118, 118, 106; 48 rows x 32 heads, a
// quarter full, 55, 41, 44; 4 x 16 rows over 3501 42, 42, 45; own keys first 135, 50, 42; with two units a warp 124, 41, 55).  What is estimated is the count of splits alone, at half full caches.
struct PxStep { int own_ctas, own_splits, splits; };
static int px_own_splits(long items) {                                 // parts that give every warp of all SMs one
  const long s = (8l * PX_SMS + items - 1) / items;
  return (int)(s < 1 ? 1 : (s > PX_MAX_OWN ? PX_MAX_OWN : s));
}
// Up to eight queries of a (group, key head): they are rows of one mma.sync operand, and a warp per part of the keys moves them as fast as an SM can take them, where a tile
// of 128 rows for tcgen05 would be all but empty.  Not where a few heads have long prefixes: one warp's part is then long, or the parts many.  us in a graph, tiles and
// this: 8 rows x 32 heads with keys of their own over 1000 17.2, 11.8, over 4000 27, 18; 5 groups of 2 over 6070 132, 100; 8 groups of 2 rows, 8 key heads, over 1000 19.6, 13.0; one
// such group over 100 10.0, 9.5, over 4000 13.2, 14.1; one key head over 19074 13, 17.
static bool px_rows(int B, int groups, int nkv, int G, int P) { return B / groups * G <= 8 && (groups * nkv >= 16 || P <= 512); }
// parts of 64 keys or more, at most one for every warp of the SMs
static int px_rows_splits(int groups, int nkv, int P) {
  const int most = (8 * PX_SMS + groups * nkv - 1) / (groups * nkv), by_keys = (P + 63) / 64;
  const int s = most < by_keys ? most : by_keys;
  return s > PX_MAX_SPLITS ? PX_MAX_SPLITS : s;
}
static PxStep px_step(int B, int groups, int nkv, int G, int hd, int P, int T) {
  PxStep r;
  const long items = (long)B * nkv, queries = (long)(B / groups) * G;
  const int most = px_own_splits(items), by_keys = (T + 127) / 128;
  r.own_splits = most < by_keys ? most : by_keys;
  r.own_ctas = (int)((items * r.own_splits + 7) / 8);
  if (px_rows(B, groups, nkv, G, P)) {
    // us: 3 in and out of a unit, 13 KB/us of keys for a warp; the rounds of CTAs that all units make, half of the longest unit, the parts to join
    const float heads = (float)groups * nkv, own = (float)items * r.own_splits, warps = 8.f * PX_SMS, key = (float)hd * 4.f / 13e3f;
    const float own_us = 3.f + (float)T * 0.5f / (float)r.own_splits * key;
    const int most = px_rows_splits(groups, nkv, P);
    float best = 0.f;
    for (int n = 1; n <= most; ++n) {
      const float us = 3.f + (float)P / (float)n * key, units = heads * n + own;
      const float c = (own * own_us + heads * n * us) / warps + 0.6f * fmaxf(us, own_us) + 1.3f * ceilf(units / warps) + 0.06f * n;
      if (best == 0.f || c < best) { best = c; r.splits = n; }
    }
    r.own_ctas = (int)((items * r.own_splits + (long)groups * nkv * r.splits + 7) / 8);
    return r;
  }
  // us: 3 in and out of a unit, 55 KB/us of own keys for the 8 warps of an SM (what one SM draws under load); 0.9 a tile of shared keys and 2 for two tiles of
  // queries (1.8 in 96 rows over 32768; splits by 1.25, 1.45, 1.7, this, 2.4: 64 rows x 32 heads over 4096 32, 30.5, 29, 26.4, 26.4; 40 over 16000 -, 42.7, 42.6, 40.6, 44.5; 2 x 48 over 8192 -, 51,
  // 51, 49, 49.3), 8 in and out of a CTA
  const float unit = 3.f + (float)T * 0.5f / (float)r.own_splits * (float)hd * 4.f * 8.f / 55e3f, tile = queries > PX_BM ? 2.0f : 0.9f;
  const int tiles = (P + PX_BN - 1) / PX_BN, cap = px_splits(queries, groups, nkv, P);       // (what the scratch is sized for)
  const bool half = queries > PX_BM && (queries % (2 * PX_BM) <= PX_BM && queries % (2 * PX_BM) != 0);
  const float heads = (float)(groups * nkv), work = heads * ((float)px_tiles(queries) - (half ? 0.22f : 0.f)) * (float)tiles * tile + (float)r.own_ctas * unit;
  float best = 0.f;
  r.splits = 1;
  for (int s = 1; s <= cap && (s == 1 || 2 * s <= tiles); ++s) {
    const float ctas = heads * (float)px_tiles(queries) * s, cta = (float)((tiles + s - 1) / s) * tile + 8.f;
    const float us = fmaxf(cta, (work + 8.f * ctas) / PX_SMS + (ctas <= PX_SMS ? 0.5f * unit : 0.4f * cta)) + (float)queries * heads * s * 3e-4f;
    if (best == 0.f || us < best) { best = us; r.splits = s; }
  }
  return r;
}

// Prompts of few tokens, own keys by a warp per (token, key head): their time in tiles of keys, 5 us in and out of 8 units.
static float px_few(int B, int S, int nkv, float keys) { return (float)B * S * nkv / (8.f * PX_SMS) * (5.6f + keys / 12.f) + 1.f; }

// S tokens per row.  Both sets of keys in one launch, every row's queries in tiles of their own, in `splits`; or the shared keys for all rows of a group together, in
// `splits`, and the own keys (taken to be the call's own tokens) in a second launch, in tiles or by warps.
struct PxPrompt { bool both; int splits; };
static PxPrompt px_prompt(int B, int S, int groups, int nkv, int G, int P) {
  const long queries = (long)(B / groups) * S * G, rows = (long)B * S * G * nkv;
  const float own = (float)S / PX_BN, shared = (float)P / PX_BN, join = 4e-4f * (float)rows;
  PxPrompt r{false, 1};
  float least;
  r.splits = px_splits(queries, groups, nkv, P, true, &least);
  least += fminf(px_rounds((long)S * G, B, nkv, 1, own, true), px_few(B, S, nkv, (float)S)) + join + 3.f;
  for (int s = 1; s <= 4; ++s) {
    const float c = px_rounds((long)S * G, B, nkv, s, (shared + own) / s, true) + (s > 1 ? s * join + 3.f : 0.f);
    if (c < least) { least = c; r = PxPrompt{true, s}; }
  }
  return r;
}

static size_t px_part_bytes(long tokens, int nh, int hd, int splits) { return (size_t)tokens * nh * splits * (hd + 2) * sizeof(float); }

}  // namespace jl

using namespace jl;

extern "C" JL_API size_t jl_prefix_attn_scratch_bytes(int B, int S, int groups, int nh, int nkv, int hd, int prefix) {
  if (B < 1 || S < 1 || groups < 1 || B % groups != 0 || nkv < 1 || nh % nkv != 0 || prefix < 0) return 0;
  const int G = nh / nkv;
  const PxPrompt plan = px_prompt(B, S, groups, nkv, G, prefix);
  int parts = plan.both ? (plan.splits > 1 ? plan.splits : 0) : plan.splits + 1;
  if (S == 1) {                                                        // either form of one token
    const int step = (px_rows(B, groups, nkv, G, prefix) ? px_rows_splits(groups, nkv, prefix) : px_splits((long)(B / groups) * G, groups, nkv, prefix)) + px_own_splits((long)B * nkv);
    parts = parts > step ? parts : step;
  }
  if (parts == 0) return 16;                                           // (nothing is left in between; never nothing)
  return px_part_bytes((long)B * S, nh, hd, parts);
}

static int px_check(const char* who, int B, int S, int groups, int nh, int nkv, int hd, int P, int T, const void* scratch, size_t scratch_bytes, const void* const* aligned,
                    int n_aligned) {
  JL_CHECK_ARG(hd == 128 || hd == 64, "%s: head_dim=%d (64 and 128 are built)", who, hd);
  JL_CHECK_ARG(nkv > 0 && nh % nkv == 0 && (nh / nkv == 1 || nh / nkv == 2 || nh / nkv == 4 || nh / nkv == 8),
               "%s: nh=%d, nkv=%d: 1, 2, 4 or 8 query heads per key head are built", who, nh, nkv);
  JL_CHECK_ARG(B >= 0 && S >= 0 && groups > 0 && B % groups == 0, "%s: %d rows of %d tokens in %d groups", who, B, S, groups);
  JL_CHECK_ARG(P >= 1 && T >= 1, "%s: caches of %d and %d slots", who, P, T);
  JL_CHECK_ARG((long)B * nkv <= 65535l * 64 && nkv <= 65535 && B <= 65535, "%s: %d rows, %d key heads", who, B, nkv);
  JL_CHECK_ARG(scratch != nullptr && scratch_bytes >= jl_prefix_attn_scratch_bytes(B, S, groups, nh, nkv, hd, P), "%s: scratch of %zu bytes, %zu are needed", who,
               scratch_bytes, jl_prefix_attn_scratch_bytes(B, S, groups, nh, nkv, hd, P));
  for (int i = 0; i < n_aligned; ++i) JL_CHECK_ARG((uintptr_t)aligned[i] % 16 == 0, "%s: tensors start at 16-byte boundaries", who);
  return JL_OK;
}

extern "C" JL_API int jl_decode_attn_prefix(const void* qkv, const void* prefix_k, const void* prefix_v, void* k_cache, void* v_cache, const float* cos_t,
                                            const float* sin_t, const int* cache_len, const int* pad_left, const int* prefix_len, const int* prefix_pad,
                                            void* scratch, size_t scratch_bytes, void* out, int B, int groups, int nh, int nkv, int hd, int P, int T, int max_pos,
                                            float scale, void* stream) {
  if (B == 0) return JL_OK;
  const void* aligned[] = {qkv, prefix_k, prefix_v, k_cache, v_cache, cos_t, sin_t, out, scratch};
  const int rc0 = px_check("jl_decode_attn_prefix", B, 1, groups, nh, nkv, hd, P, T, scratch, scratch_bytes, aligned, 9);
  if (rc0) return rc0;
  JL_CHECK_ARG(cache_len != nullptr && max_pos >= 1, "jl_decode_attn_prefix: the slot of the new token and its tables are required");
  const int G = nh / nkv, rows = B / groups;
  JL_CHECK_ARG((long)B * nh < (1l << 26), "jl_decode_attn_prefix: %d rows of %d heads", B, nh);
  const PxStep plan = px_step(B, groups, nkv, G, hd, P, T);
  PxParams p{};
  p.q = (const __nv_bfloat16*)qkv; p.ldq = (nh + 2 * nkv) * hd;
  p.k_cache = (__nv_bfloat16*)k_cache; p.v_cache = (__nv_bfloat16*)v_cache;
  p.cos_t = cos_t; p.sin_t = sin_t; p.max_pos = max_pos; p.cache_len = cache_len;
  p.prefix_len = prefix_len; p.prefix_pad = prefix_pad; p.pad_left = pad_left;
  p.S = 1; p.B = B; p.rows = rows; p.nh = nh; p.nkv = nkv; p.gs = G == 1 ? 0 : (G == 2 ? 1 : (G == 4 ? 2 : 3)); p.P = P; p.T = T;
  p.shared = 1; p.partial = 1;
  p.own_ctas = plan.own_ctas; p.own_splits = plan.own_splits; p.splits = plan.splits; p.parts = plan.splits + plan.own_splits;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.o_part = (float*)scratch;
  p.ml_part = (float2*)(p.o_part + (size_t)B * nh * p.parts * hd);
  int rc;
  if (px_rows(B, groups, nkv, G, P)) {
    p.prefix_k = (const __nv_bfloat16*)prefix_k; p.prefix_v = (const __nv_bfloat16*)prefix_v;
    rc = hd == 128 ? px_warps_launch<128, true>(p, (cudaStream_t)stream) : px_warps_launch<64, true>(p, (cudaStream_t)stream);
  } else {
    CUtensorMap pk, pv;
    rc = make_tmap_3d_bf16(&pk, prefix_k, (uint64_t)groups * nkv, P, hd, (uint64_t)P * hd, hd, PX_BN);
    if (rc == JL_OK) rc = make_tmap_3d_bf16(&pv, prefix_v, (uint64_t)groups * nkv, P, hd, (uint64_t)P * hd, hd, PX_BN);
    if (rc == JL_OK) rc = px_dispatch(p, (long)rows * G, groups, true, hd, pk, pv, pk, pv, (cudaStream_t)stream);
  }
  if (rc != JL_OK) return rc;
  return px_join(p, (__nv_bfloat16*)out, B * nh, hd, -1, (cudaStream_t)stream);
}

extern "C" JL_API int jl_prefill_attn_prefix(const void* q, const void* prefix_k, const void* prefix_v, const void* k_cache, const void* v_cache,
                                             const int* pad_left, const int* prefix_len, const int* prefix_pad, void* scratch, size_t scratch_bytes, void* out,
                                             int B, int S, int groups, int nh, int nkv, int hd, int P, int T, int start, float scale, void* stream) {
  if (B == 0 || S == 0) return JL_OK;
  const void* aligned[] = {q, prefix_k, prefix_v, k_cache, v_cache, out, scratch};
  int rc = px_check("jl_prefill_attn_prefix", B, S, groups, nh, nkv, hd, P, T, scratch, scratch_bytes, aligned, 7);
  if (rc) return rc;
  JL_CHECK_ARG(start >= 0 && start <= T - S, "jl_prefill_attn_prefix: start=%d + S=%d exceeds cache capacity %d", start, S, T);
  const int G = nh / nkv, rows = B / groups;
  JL_CHECK_ARG((long)B * S * nh < (1l << 31), "jl_prefill_attn_prefix: %d rows of %d tokens of %d heads", B, S, nh);
  CUtensorMap pk, pv, ok, ov;
  rc = make_tmap_3d_bf16(&pk, prefix_k, (uint64_t)groups * nkv, P, hd, (uint64_t)P * hd, hd, PX_BN);
  if (rc == JL_OK) rc = make_tmap_3d_bf16(&pv, prefix_v, (uint64_t)groups * nkv, P, hd, (uint64_t)P * hd, hd, PX_BN);
  if (rc == JL_OK) rc = make_tmap_3d_bf16(&ok, k_cache, (uint64_t)B * nkv, T, hd, (uint64_t)T * hd, hd, PX_BN);
  if (rc == JL_OK) rc = make_tmap_3d_bf16(&ov, v_cache, (uint64_t)B * nkv, T, hd, (uint64_t)T * hd, hd, PX_BN);
  if (rc != JL_OK) return rc;
  PxParams p{};
  p.q = (const __nv_bfloat16*)q; p.ldq = nh * hd;
  p.prefix_len = prefix_len; p.prefix_pad = prefix_pad; p.pad_left = pad_left;
  p.out = (__nv_bfloat16*)out;
  p.S = S; p.rows = rows; p.nh = nh; p.nkv = nkv; p.gs = G == 1 ? 0 : (G == 2 ? 1 : (G == 4 ? 2 : 3)); p.P = P; p.T = T; p.start = start;
  p.scale_log2 = scale * 1.4426950408889634f;
  const PxPrompt plan = px_prompt(B, S, groups, nkv, G, P);
  p.splits = plan.splits;
  p.parts = plan.both ? plan.splits : plan.splits + 1;
  p.o_part = (float*)scratch;
  p.ml_part = (float2*)(p.o_part + (size_t)B * S * nh * p.parts * hd);
  if (plan.both) {
    p.shared = p.own = 1;
    p.partial = p.splits > 1;
    rc = px_dispatch(p, (long)S * G, B, false, hd, pk, pv, ok, ov, (cudaStream_t)stream);
    if (rc != JL_OK || !p.partial) return rc;
    return px_join(p, (__nv_bfloat16*)out, B * S * nh, hd, -1, (cudaStream_t)stream);
  }
  p.shared = p.partial = 1;
  const long units = (long)B * S * nkv;
  const bool few = units < (1l << 30) && px_few(B, S, nkv, (float)(start + S)) < px_rounds((long)S * G, B, nkv, 1, (float)(start + S) / PX_BN, true);
  rc = px_dispatch(p, (long)rows * S * G, groups, false, hd, pk, pv, ok, ov, (cudaStream_t)stream);
  if (rc != JL_OK) return rc;
  if (few) {
    p.k_cache = (__nv_bfloat16*)k_cache; p.v_cache = (__nv_bfloat16*)v_cache;            // (read only)
    p.B = B; p.own_splits = 1; p.own_ctas = (int)((units + 7) / 8);
    rc = hd == 128 ? px_warps_launch<128, false>(p, (cudaStream_t)stream) : px_warps_launch<64, false>(p, (cudaStream_t)stream);
    return rc != JL_OK ? rc : px_join(p, (__nv_bfloat16*)out, B * S * nh, hd, p.splits, (cudaStream_t)stream);
  }
  p.shared = 0; p.own = 1; p.part0 = p.splits; p.splits = 1;
  rc = px_dispatch(p, (long)S * G, B, false, hd, pk, pv, ok, ov, (cudaStream_t)stream);
  if (rc != JL_OK) return rc;
  return px_join(p, (__nv_bfloat16*)out, B * S * nh, hd, p.part0, (cudaStream_t)stream);
}
