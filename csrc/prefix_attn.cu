// Attention of a batch whose rows share keys: a prompt with several answers, a document with many questions.
//
//   out(b, s, h) = softmax_j (q · k_j / sqrt(d)) v_j   over the keys [prefix_pad, prefix_len) of the row's group, the same for all its rows, and the
//                  row's own keys [pad_left, slot of the query]
//
// The shared keys are read once for all rows: the queries of a group, every row's tokens and the G query heads of a key head, are the rows of one
// matrix [rows · S · G, d] per (group, key head), cut into tiles of 128 for tcgen05.  With running statistics a softmax over two sets of keys
// is a join of two triples (reference exponent m, sum l, weighted values o):  M = max(m1, m2),  o = o1 2^(m1 - M) + o2 2^(m2 - M),  l likewise.
//   * one token per row (jl_decode_attn_prefix): shared keys in tiles of queries here, cut into splits over the SMs, partial triples in fp32; then the
//     rows' own keys in the one-token kernel (decode_attn_fused.cu), which appends the new key and joins;
//   * S tokens per row (jl_prefill_attn_prefix): the same for the shared keys, then a second launch of this kernel over every row's own keys, causal, that
//     joins in its last step; or one launch over both sets, tile after tile, where a row's queries fill tiles by themselves.
//
// One CTA owns a tile of 128 queries of one key head, as in flash_prefill.cu: a warp asks for K and V tiles of 64 keys (TMA, 128-byte swizzle), a warp
// issues S = Q·Kᵀ into one of two score tiles in TMEM and O += P·V with P read from TMEM, four warps hold one query row per thread: one pass over 64
// scores in registers, exponentials in base 2 against a reference that is raised only when it has grown by 2^8.
// Queries go to shared memory by hand: rows of different tokens and heads follow each other in a tile, and the one-token form rotates them on the way.
// A rotated query is kept as two bfloat16 numbers, hi + lo (two products into the same scores): rounded to one, a score of size s would be off by
// s 2^-9 and the result by as much again as its own rounding.  Probabilities are rounded to bfloat16 (2^-9 of each weight, sums in fp32).
// Slots that hold no key may hold anything: their scores are masked, and their value rows are cleared in shared memory, because a weight of zero
// times a NaN is a NaN.
#include <atomic>

#include "jllama_b200.h"
#include "prefix_attn.cuh"
#include "tcgen05.cuh"

namespace jl {

constexpr int PX_BM = 128, PX_BN = 64, PX_THREADS = 192;
constexpr float PX_RESCALE = 8.0f;                                 // log2 units
constexpr uint32_t PX_BARS = 256;                                  // barriers and the address of the TMEM columns

template <int HD> struct PxTile {
  static constexpr int HALVES = HD / 64;
  static constexpr uint32_t Q_HALF = PX_BM * 128, Q = HALVES * Q_HALF;       // bytes
  static constexpr uint32_t KV_HALF = PX_BN * 128, SLOT = HALVES * KV_HALF;
  static constexpr uint32_t TMEM_COLS = 256;
};

struct PxParams {
  const __nv_bfloat16* q; int ldq;  // token t, head h at q + t · ldq + h · HD
  const float* cos_t; const float* sin_t; int max_pos; const int* cache_len;     // ROTATE: tables and the slot of the new token
  const int* prefix_len; const int* prefix_pad; const int* pad_left;
  __nv_bfloat16* out;
  float* o_part; float2* ml_part;   // [tokens · nh][splits]: written (partial) or joined (own keys behind a launch over the shared ones)
  int S, rows, nh, nkv, P, T, start;
  int shared, own, partial;         // which keys this launch visits; whether it leaves partial triples or the result
  int smem;                         // bytes of dynamic shared memory
  int splits, join, slots;          // splits of the shared keys in this launch; triples per (token, head) that the last step joins; tiles of the ring
  float scale_log2;
};

template <int HD, bool ROTATE>
__global__ void __launch_bounds__(256, 2)        // 256: caps registers at 128, so that two six-warp CTAs (allocated as eight) fit
prefix_attn_kernel(const __grid_constant__ CUtensorMap tm_pk, const __grid_constant__ CUtensorMap tm_pv,
                   const __grid_constant__ CUtensorMap tm_ok, const __grid_constant__ CUtensorMap tm_ov, const PxParams p) {
  using Tile = PxTile<HD>;
  constexpr int HALVES = Tile::HALVES;
  constexpr int NQ = ROTATE ? 2 : 1;             // hi, lo
  extern __shared__ __align__(1024) uint8_t px_smem[];
  const uint32_t raw = tc::smem_u32(px_smem);
  const uint32_t base = (raw + 1023u) & ~1023u;  // the 128-byte swizzle counts rows from 1024-byte boundaries
  const uint32_t sQ = base, ring = base + NQ * Tile::Q;
  const uint32_t bars = ring + p.slots * Tile::SLOT;
  const uint32_t q_full = bars, p_full = bars + 8, o_full = bars + 16;
  auto s_full = [&](int s) { return bars + 24 + 8u * s; };
  auto slot_full = [&](int s) { return bars + 48 + 16u * s; };
  auto slot_empty = [&](int s) { return bars + 56 + 16u * s; };
  const uint32_t tmem_slot = bars + 40;
  if (bars + PX_BARS > raw + p.smem) __trap();   // dynamic shared memory less aligned than budgeted
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(px_smem + (tmem_slot - raw));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.nh / p.nkv;
  // z: group (shared keys alone) or row; y: key head; x: query tile, and split for partial results
  const int kvh = blockIdx.y, z = blockIdx.z;
  const int qt = (int)(gridDim.x / p.splits) - 1 - (int)blockIdx.x / p.splits;      // longest first
  const int split = blockIdx.x % p.splits;
  const int unit_tokens = p.own ? p.S : p.rows * p.S;             // tokens whose queries this launch packs together
  const int token0 = z * unit_tokens;
  const int q0 = qt * PX_BM, n_rows = min(PX_BM, unit_tokens * G - q0);
  const int group = p.own ? z / p.rows : z;

  if (warp == 0 && lane == 0) {
    if (p.shared) { tc::prefetch_tensormap(&tm_pk); tc::prefetch_tensormap(&tm_pv); }
    if (p.own) { tc::prefetch_tensormap(&tm_ok); tc::prefetch_tensormap(&tm_ov); }
  }
  if (warp == 1 && lane == 0) {
    tc::mbar_init(q_full, 4); tc::mbar_init(p_full, 4); tc::mbar_init(o_full, 1);
    tc::mbar_init(s_full(0), 1); tc::mbar_init(s_full(1), 1);
    for (int s = 0; s < p.slots; ++s) { tc::mbar_init(slot_full(s), 1); tc::mbar_init(slot_empty(s), 1); }
    tc::fence_barrier_init();
  }
  if (warp == 0) tc::tmem_alloc(tmem_slot, Tile::TMEM_COLS);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot_ptr;
  auto tS = [&](int j) { return tmem + (uint32_t)(j & 1) * 64u; };     // score tile j, afterwards its probabilities
  const uint32_t tO = tmem + 128;

  pdl_wait();
  pdl_launch_dependents();

  // shared keys [s_lo, s_hi) of this CTA, own keys [o_lo, o_hi)
  int s_lo = 0, s_hi = 0, o_lo = 0, o_hi = 0;
  const int g_lo = p.prefix_pad ? max(p.prefix_pad[group], 0) : 0;
  const int g_hi = p.prefix_len ? min(p.prefix_len[group], p.P) : p.P;
  if (p.shared) {
    const int n = max(g_hi - g_lo, 0);
    const int chunk = ((n + p.splits - 1) / p.splits + PX_BN - 1) / PX_BN * PX_BN;
    s_lo = g_lo + min(split * chunk, n);
    s_hi = g_lo + min((split + 1) * chunk, n);
  }
  const int pad = p.pad_left ? max(p.pad_left[p.own ? z : 0], 0) : 0;  // (own keys only; the one-token form reads the rows' pads itself)
  if (p.own) {
    o_lo = pad;
    o_hi = max(p.start + (q0 + n_rows - 1) / G + 1, o_lo);             // slot of the tile's last token: its last key
  }
  const int n_shared = (s_hi - s_lo + PX_BN - 1) / PX_BN, n_tiles = n_shared + (o_hi - o_lo + PX_BN - 1) / PX_BN;

  if (warp == 0) {
    if (lane == 0) {
      int sl = 0;
      uint32_t ph = 1;
      for (int idx = 0; idx < 2 * n_tiles; ++idx) {                    // K_0, V_0, K_1, V_1, ...
        const int j = idx >> 1;
        const bool mine = j >= n_shared;
        const CUtensorMap* m = (idx & 1) ? (mine ? &tm_ov : &tm_pv) : (mine ? &tm_ok : &tm_pk);
        const int key0 = mine ? o_lo + (j - n_shared) * PX_BN : s_lo + j * PX_BN;
        const int head = (mine ? z : group) * p.nkv + kvh;
        tc::mbar_wait(slot_empty(sl), ph);
        tc::mbar_expect_tx(slot_full(sl), Tile::SLOT);
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          tc::tma_load_3d(ring + sl * Tile::SLOT + h * Tile::KV_HALF, m, slot_full(sl), 64 * h, key0, head, tc::EVICT_NORMAL);
        if (++sl == p.slots) { sl = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    // the whole warp walks the loop, one elected lane issues; descriptors are advanced by their address field (flash_prefill.cu)
    constexpr uint32_t IDESC_S = tc::idesc_bf16_f32(PX_BM, PX_BN, false, false);
    constexpr uint32_t IDESC_O = tc::idesc_bf16_f32(PX_BM, HD, false, true);        // B = V is MN-major
    const uint64_t dQ = tc::smem_desc_kmajor_sw128(sQ);
    const uint64_t dK0 = tc::smem_desc_kmajor_sw128(ring);
    const uint64_t dV0 = tc::smem_desc_mnmajor_sw128(ring, Tile::KV_HALF, 1024);
    int sl = 0;                                                        // slot of the next K or V tile in issue order K_0, K_1, V_0, K_2, V_1, ...
    auto at = [&](int idx, uint32_t* phase) {                          // where tile number idx of the ring lies
      const int use = idx / p.slots;
      *phase = use & 1;
      return idx - use * p.slots;
    };
    auto issue_s = [&](int j) {
      uint32_t ph;
      sl = at(2 * j, &ph);
      tc::mbar_wait(slot_full(sl), ph);
      tc::fence_after_sync();
      if (tc::elect_one()) {
        const uint64_t dK = dK0 + (uint64_t)sl * (Tile::SLOT >> 4);
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            tc::mma_ss(tS(j), dQ + (uint64_t)((n * Tile::Q + (k >> 2) * Tile::Q_HALF + (k & 3) * 32) >> 4),
                       dK + (uint64_t)(((k >> 2) * Tile::KV_HALF + (k & 3) * 32) >> 4), IDESC_S, n != 0 || k != 0);
        tc::mma_commit(s_full(j & 1));
        tc::mma_commit(slot_empty(sl));
      }
      __syncwarp();
    };
    if (n_tiles > 0) {
      tc::mbar_wait(q_full, 0);
      tc::fence_after_sync();
      issue_s(0);
    }
    for (int j = 0; j < n_tiles; ++j) {
      if (j + 1 < n_tiles) issue_s(j + 1);                             // the tensor core forms S_{j+1} during softmax_j
      uint32_t ph;
      sl = at(2 * j + 1, &ph);
      tc::mbar_wait(slot_full(sl), ph);
      const int left = j < n_shared ? s_hi - s_lo - j * PX_BN : o_hi - o_lo - (j - n_shared) * PX_BN;
      if (left < PX_BN) {                                              // value rows that hold no key
        for (int i = lane; i < (PX_BN - left) * 8 * HALVES; i += 32) {
          const int r = left + i / (8 * HALVES), c = i % (8 * HALVES);
          const uint32_t a = ring + sl * Tile::SLOT + (c >> 3) * Tile::KV_HALF + r * 128 + (c & 7) * 16;
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      tc::mbar_wait(p_full, j & 1);
      tc::fence_after_sync();
      if (tc::elect_one()) {
        const uint64_t dV = dV0 + (uint64_t)sl * (Tile::SLOT >> 4);
#pragma unroll
        for (int k = 0; k < PX_BN / 16; ++k)                           // A = P_j in TMEM: 16 keys = 8 columns of packed pairs
          tc::mma_ts(tO, tS(j) + k * 8, dV + (uint64_t)((k * 2048) >> 4), IDESC_O, j != 0 || k != 0);
        tc::mma_commit(o_full);
        tc::mma_commit(slot_empty(sl));
      }
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3;                                      // TMEM lane quadrant of this warp
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    // ---- queries: the warp's 32 rows, 16 bytes per lane and step
    constexpr int CH = HD / 8, RPS = 32 / CH;                          // 16-byte chunks of a row, rows of a step
    const int ch = lane % CH;
    if (n_tiles > 0) {
#pragma unroll 4
      for (int i = 0; i < CH; ++i) {
        const int r = quarter * 32 + i * RPS + lane / CH;
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (r < n_rows) {
          const int token = token0 + (q0 + r) / G, h = kvh * G + (q0 + r) % G;
          hi = *reinterpret_cast<const uint4*>(p.q + (size_t)token * p.ldq + (size_t)h * HD + 8 * ch);
          if constexpr (ROTATE) {
            int pos = max(g_hi - g_lo, 0) + min(*p.cache_len, p.T) - (p.pad_left ? p.pad_left[token] : 0);
            pos = pos < 0 ? 0 : (pos >= p.max_pos ? p.max_pos - 1 : pos);
            const float4 c4 = __ldg(reinterpret_cast<const float4*>(p.cos_t) + (size_t)pos * CH + ch);
            const float4 s4 = __ldg(reinterpret_cast<const float4*>(p.sin_t) + (size_t)pos * CH + ch);
            const float cs[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
            const uint32_t w[4] = {hi.x, hi.y, hi.z, hi.w};
            uint32_t a[4], b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float re = bf16_lo(w[e]), im = bf16_hi(w[e]);
              const float u = re * cs[e] - im * sn[e], v = re * sn[e] + im * cs[e];
              a[e] = pack_bf16(u, v);
              b[e] = pack_bf16(u - bf16_lo(a[e]), v - bf16_hi(a[e]));
            }
            hi = make_uint4(a[0], a[1], a[2], a[3]);
            lo = make_uint4(b[0], b[1], b[2], b[3]);
          }
        }
        const uint32_t dst = sQ + (ch >> 3) * Tile::Q_HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w) : "memory");
        if constexpr (ROTATE)
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + Tile::Q), "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full);
    }

    const int r = quarter * 32 + lane;                                 // this thread's query
    const bool row_on = r < n_rows;
    const int slot = p.own ? p.start + (q0 + min(r, n_rows - 1)) / G : 0;             // of the query's own key
    const int slot_warp = p.own ? p.start + (q0 + min(quarter * 32, n_rows - 1)) / G : 0;      // the smallest of the warp
    float m_ref = -INFINITY, l_run = 0.f;
    for (int j = 0; j < n_tiles; ++j) {
      const bool mine = j >= n_shared;
      const int key0 = mine ? o_lo + (j - n_shared) * PX_BN : s_lo + j * PX_BN;
      const int end = mine ? slot + 1 : s_hi;                          // first key that this row does not see
      const bool need_mask = key0 + PX_BN > (mine ? slot_warp + 1 : s_hi);       // warp-uniform
      tc::mbar_wait(s_full(j & 1), (j >> 1) & 1);
      tc::fence_after_sync();
      uint32_t v0[32], v1[32];
      tc::tmem_ld32(tS(j) + lane_off, v0);
      tc::tmem_ld32(tS(j) + lane_off + 32, v1);
      tc::tmem_ld_wait();
      if (need_mask) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (key0 + i >= end) v0[i] = 0xff800000u;                    // -inf
          if (key0 + 32 + i >= end) v1[i] = 0xff800000u;
        }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 32; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], fmaxf(__uint_as_float(v0[i]), __uint_as_float(v1[i])));
      const float t = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
      const bool need = t > m_ref + PX_RESCALE || (m_ref == -INFINITY && t > -INFINITY);
      if (j == 0) {
        m_ref = t;
      } else if (__any_sync(0xffffffffu, need)) {
        const float factor = need ? exp2f(m_ref - t) : 1.0f;           // m_ref = -inf: 0 (O and l are 0 there)
        tc::mbar_wait(o_full, (j - 1) & 1);                            // O at rest
        tc::fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tc::tmem_ld32(tO + lane_off + c * 32, o);
          tc::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
          tc::tmem_st32(tO + lane_off + c * 32, o);
        }
        tc::tmem_st_wait();
        l_run *= factor;
        if (need) m_ref = t;
      }
      const float m_safe = m_ref == -INFINITY ? 0.f : m_ref;
      float psum = 0.f;
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float a0 = exp2f(fmaf(__uint_as_float(v0[2 * i]), p.scale_log2, -m_safe));
        const float a1 = exp2f(fmaf(__uint_as_float(v0[2 * i + 1]), p.scale_log2, -m_safe));
        const float b0 = exp2f(fmaf(__uint_as_float(v1[2 * i]), p.scale_log2, -m_safe));
        const float b1 = exp2f(fmaf(__uint_as_float(v1[2 * i + 1]), p.scale_log2, -m_safe));
        psum += (a0 + a1) + (b0 + b1);
        w[i] = pack_bf16(a0, a1);
        w[16 + i] = pack_bf16(b0, b1);
      }
      tc::tmem_st32(tS(j) + lane_off, w);                              // keys 2c, 2c + 1 of this row: 32-bit column c
      tc::tmem_st_wait();
      l_run += psum;
      // at most one phase of p_full outstanding: P·V_{j-1} done proves that the MMA warp has seen phase j - 1 (flash_prefill.cu)
      if (j > 0) tc::mbar_wait(o_full, (j - 1) & 1);
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_full);
    }
    if (n_tiles > 0) {
      tc::mbar_wait(o_full, (n_tiles - 1) & 1);
      tc::fence_after_sync();
    }
    const int token = token0 + (q0 + min(r, n_rows - 1)) / G, h = kvh * G + (q0 + min(r, n_rows - 1)) % G;
    const size_t th = (size_t)token * p.nh + h;
    if (p.partial) {
      const size_t part = th * p.splits + split;
      if (row_on) p.ml_part[part] = make_float2(m_ref, l_run);
      float4* dst = reinterpret_cast<float4*>(p.o_part + part * HD);
      if (n_tiles > 0) {
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tc::tmem_ld32(tO + lane_off + c * 32, o);
          tc::tmem_ld_wait();
          if (row_on) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[8 * c + i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
          }
        }
      }
    } else {
      // ---- join with the partial triples of the shared keys (none when this launch visited them), normalise, store the row
      const int n_parts = p.join;
      const bool seen = row_on && slot >= pad;                         // a query in front of its row's first token is padding: zeros
      float M = l_run != 0.f ? m_ref : -INFINITY;                      // (a sum of zero: no keys; NaN stays NaN)
      const float2* ml = p.ml_part + th * n_parts;
      if (seen)
        for (int s = 0; s < n_parts; ++s) {
          const float2 v = __ldcg(ml + s);
          if (v.y != 0.f) M = fmaxf(M, v.x);
        }
      const float Ms = M == -INFINITY ? 0.f : M;
      const float f0 = l_run != 0.f ? exp2f(m_ref - Ms) : 0.f;
      float L = l_run * f0;
      if (seen)
        for (int s = 0; s < n_parts; ++s) {
          const float2 v = __ldcg(ml + s);
          if (v.y != 0.f) L += v.y * exp2f(v.x - Ms);
        }
      const float inv = seen && L != 0.f ? 1.0f / L : 0.f;
      uint4* dst = reinterpret_cast<uint4*>(p.out + th * HD);
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        if (n_tiles > 0) {
          tc::tmem_ld32(tO + lane_off + c * 32, o);
          tc::tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = f0 != 0.f ? __float_as_uint(__uint_as_float(o[i]) * f0) : 0u;
        if (seen) {
          for (int s = 0; s < n_parts; ++s) {
            const float2 v = __ldcg(ml + s);
            if (v.y == 0.f) continue;
            const float f = exp2f(v.x - Ms);
            const float4* src = reinterpret_cast<const float4*>(p.o_part + (th * n_parts + s) * HD + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 x = __ldcg(src + i);
              o[4 * i] = __float_as_uint(fmaf(x.x, f, __uint_as_float(o[4 * i])));
              o[4 * i + 1] = __float_as_uint(fmaf(x.y, f, __uint_as_float(o[4 * i + 1])));
              o[4 * i + 2] = __float_as_uint(fmaf(x.z, f, __uint_as_float(o[4 * i + 2])));
              o[4 * i + 3] = __float_as_uint(fmaf(x.w, f, __uint_as_float(o[4 * i + 3])));
            }
          }
        }
        if (row_on) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            auto v = [&](int e) { return seen ? __uint_as_float(o[8 * i + e]) * inv : 0.f; };
            dst[c * 4 + i] = make_uint4(pack_bf16(v(0), v(1)), pack_bf16(v(2), v(3)), pack_bf16(v(4), v(5)), pack_bf16(v(6), v(7)));
          }
        }
      }
    }
    tc::fence_before_sync();
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, Tile::TMEM_COLS);
}

template <int HD, bool ROTATE>
static int px_launch(PxParams p, dim3 grid, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& ok, const CUtensorMap& ov, cudaStream_t st) {
  using Tile = PxTile<HD>;
  // slack for the alignment of the base; two rotated 128-wide CTAs fill an SM's 228 KB to the last byte with 768
  const int smem = (int)((ROTATE ? 2 : 1) * Tile::Q + p.slots * Tile::SLOT + PX_BARS + (ROTATE && HD == 128 ? 768 : 1024));
  p.smem = smem;
  // attributes belong to the device's context: set at the first call on each (bit per device; setting them twice is harmless)
  static std::atomic<uint64_t> set{0};
  int dev = 0;
  JL_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit == 0 || !(set.load(std::memory_order_acquire) & bit)) {
    JL_CUDA(cudaFuncSetAttribute(prefix_attn_kernel<HD, ROTATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    JL_CUDA(cudaFuncSetAttribute(prefix_attn_kernel<HD, ROTATE>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    set.fetch_or(bit, std::memory_order_release);
  }
  JL_CUDA(launch_pdl(prefix_attn_kernel<HD, ROTATE>, grid, dim3(PX_THREADS), (size_t)smem, st, pk, pv, ok, ov, p));
  return JL_OK;
}

static int px_dispatch(const PxParams& p, dim3 grid, bool rotate, int hd, const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& ok,
                       const CUtensorMap& ov, cudaStream_t st) {
  if (hd == 128) return rotate ? px_launch<128, true>(p, grid, pk, pv, ok, ov, st) : px_launch<128, false>(p, grid, pk, pv, ok, ov, st);
  return rotate ? px_launch<64, true>(p, grid, pk, pv, ok, ov, st) : px_launch<64, false>(p, grid, pk, pv, ok, ov, st);
}

constexpr int PX_MAX_SPLITS = 64;

// Splits of the shared keys: as many CTAs as run at once (two per SM) when that leaves every CTA two tiles of keys or more.
static int px_splits(long tokens_per_group, int groups, int nkv, int G, int prefix) {
  const long items = (tokens_per_group * G + PX_BM - 1) / PX_BM * groups * nkv;
  const long most = ((long)prefix + 2 * PX_BN - 1) / (2 * PX_BN);
  long s = 2 * 148 / (items > 0 ? items : 1);
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : (s > PX_MAX_SPLITS ? PX_MAX_SPLITS : s));
}

// Whether a row's queries fill tiles by themselves: one launch over shared and own keys.
static bool px_one_launch(int S, int G, int B, int nkv) {
  const long tiles = ((long)S * G + PX_BM - 1) / PX_BM;
  return 8l * S * G >= 7 * tiles * PX_BM && tiles * B * nkv >= 148;
}

static size_t px_part_bytes(long tokens, int nh, int hd, int splits) { return (size_t)tokens * nh * splits * (hd + 2) * sizeof(float); }
static size_t px_up(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace jl

using namespace jl;

extern "C" JL_API size_t jl_prefix_attn_scratch_bytes(int B, int S, int groups, int nh, int nkv, int hd, int prefix) {
  if (B < 1 || S < 1 || groups < 1 || B % groups != 0 || nkv < 1 || nh % nkv != 0 || prefix < 0) return 0;
  const int G = nh / nkv, splits = px_splits((long)(B / groups) * S, groups, nkv, G, prefix);
  if (S > 1 && px_one_launch(S, G, B, nkv)) return 16;             // (no partial results; never nothing)
  return px_up(S == 1 ? prefix_step_scratch_bytes(B, nh, nkv, hd) : 0) + px_part_bytes((long)B * S, nh, hd, splits);
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
  CUtensorMap pk, pv;
  int rc = make_tmap_3d_bf16(&pk, prefix_k, (uint64_t)groups * nkv, P, hd, (uint64_t)P * hd, hd, PX_BN);
  if (rc == JL_OK) rc = make_tmap_3d_bf16(&pv, prefix_v, (uint64_t)groups * nkv, P, hd, (uint64_t)P * hd, hd, PX_BN);
  if (rc != JL_OK) return rc;
  PxParams p{};
  p.q = (const __nv_bfloat16*)qkv; p.ldq = (nh + 2 * nkv) * hd;
  p.cos_t = cos_t; p.sin_t = sin_t; p.max_pos = max_pos; p.cache_len = cache_len;
  p.prefix_len = prefix_len; p.prefix_pad = prefix_pad; p.pad_left = pad_left;
  p.S = 1; p.rows = rows; p.nh = nh; p.nkv = nkv; p.P = P; p.T = T;
  p.shared = 1; p.partial = 1;
  p.splits = px_splits(rows, groups, nkv, G, P);
  p.slots = hd == 128 ? 3 : 6;
  p.scale_log2 = scale * 1.4426950408889634f;
  char* parts = (char*)scratch + px_up(prefix_step_scratch_bytes(B, nh, nkv, hd));
  p.o_part = (float*)parts;
  p.ml_part = (float2*)(p.o_part + (size_t)B * nh * p.splits * hd);
  rc = px_dispatch(p, dim3((rows * G + PX_BM - 1) / PX_BM * p.splits, nkv, groups), true, hd, pk, pv, pk, pv, (cudaStream_t)stream);
  if (rc != JL_OK) return rc;
  const PrefixStep step{(const __nv_bfloat16*)qkv, (__nv_bfloat16*)k_cache, (__nv_bfloat16*)v_cache, cos_t, sin_t, cache_len, pad_left, prefix_len, prefix_pad,
                        (__nv_bfloat16*)out, scratch, B, rows, nh, nkv, hd, P, T, max_pos, scale, {p.o_part, p.ml_part, p.splits}};
  return prefix_step_launch(step, (cudaStream_t)stream);
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
  JL_CHECK_ARG((long)rows * S * G <= (1l << 30), "jl_prefill_attn_prefix: %d rows of %d tokens share one prefix", rows, S);
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
  p.S = S; p.rows = rows; p.nh = nh; p.nkv = nkv; p.P = P; p.T = T; p.start = start;
  p.slots = hd == 128 ? 4 : 8;
  p.scale_log2 = scale * 1.4426950408889634f;
  const dim3 own_grid((S * G + PX_BM - 1) / PX_BM, nkv, B);
  p.splits = 1;
  if (px_one_launch(S, G, B, nkv)) {
    p.shared = p.own = 1;
    return px_dispatch(p, own_grid, false, hd, pk, pv, ok, ov, (cudaStream_t)stream);
  }
  const int splits = px_splits((long)rows * S, groups, nkv, G, P);
  p.o_part = (float*)((char*)scratch + px_up(S == 1 ? prefix_step_scratch_bytes(B, nh, nkv, hd) : 0));
  p.ml_part = (float2*)(p.o_part + (size_t)B * S * nh * splits * hd);
  p.shared = p.partial = 1; p.splits = splits;
  rc = px_dispatch(p, dim3((rows * S * G + PX_BM - 1) / PX_BM * splits, nkv, groups), false, hd, pk, pv, ok, ov, (cudaStream_t)stream);
  if (rc != JL_OK) return rc;
  p.shared = p.partial = 0; p.own = 1; p.splits = 1; p.join = splits;
  return px_dispatch(p, own_grid, false, hd, pk, pv, ok, ov, (cudaStream_t)stream);
}
