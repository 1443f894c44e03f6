// The rules of a request on the logits of a step: penalties for tokens that occurred, biases, a mask of allowed tokens.
//
//   x = logits[b, v]
//   v occurs in tokens[b, start_b .. len_b):               x = x > 0 ? x / r_b : x r_b                    (repetition)
//   n = occurrences in tokens[b, prompt_b .. len_b), n > 0: x = x - f_b n - p_b                           (frequency, presence)
//   entries i with bias_ids[b, i] == v:                    x = x + sum of bias[b, i]                      (summed in the order of the entries, added once)
//   bit v of allowed[b] is zero:                           x = -infinity
//
// A CTA owns a slice of one row's vocabulary and keeps one word per token of the slice in shared memory: occurrences behind the prompt in the low bits, and bits
// for "occurred", "has a bias", "has several" (whole numbers and bits: the order of the atomics does not show).  Everything it reads is asked for at once, the slice's
// logits, the row's bounds, the first tokens of its history, its first biases: a CTA's way is a chain of memory latencies.  A second table has the bias of a
// token; where there are several, the thread that was first to mark it goes through all of them in their order.  No state is kept between calls: the history is the
// sequence buffer that the decode loop writes anyway, so forks, restarts and replayed graphs need nothing.
//
// One B200, us in a graph: 96 x 128256 with 4000 tokens, 300 biases and masks 30 (3.4 TB/s; logits alone 16, the history 8, the biases 4), bound by the instructions
// issued, 66 % of the slots, some 50 a token; 17 x 128259 5.4, 1 x 32000 2.3, a launch and a chain of loads; 16-bit logits 31, 5.8, 2.4.
#include "common.cuh"
#include "jllama_b200.h"

#include <cuda_fp16.h>

namespace jl {

constexpr unsigned LR_SAID = 1u << 31, LR_BIAS = 1u << 30, LR_MORE = 1u << 29, LR_COUNT = LR_MORE - 1u;

struct RulesParams {
  const void* logits; int ld;
  float* out; int ldo;
  int V;
  const int* tokens; int ldt, T;
  const int* starts; int starts_n;                  // [B] or one for all rows (n = 1), or nullptr
  const int* lengths; int lengths_n;
  const int* prompts; int prompts_n;
  const float* rep; const float* freq; const float* pres;       // [B] or nullptr: the scalar
  float rep1, freq1, pres1;
  const int* bias_ids; const float* bias; int n_bias, ldb;
  const unsigned* allowed; int lda;
};

// TH threads with N groups of four tokens each.  Rows whose logits and results lie alike on 16-byte boundaries (8-byte ones for 16-bit logits)
// start their groups there, others load and store token by token.
template <typename T, int TH, int N>
__global__ void __launch_bounds__(TH, 1024 / TH) logit_rules_kernel(const RulesParams p) {
  constexpr int SLICE = 4 * N * TH;
  extern __shared__ __align__(16) unsigned lr_count[];
  float* lr_value = reinterpret_cast<float*>(lr_count + SLICE);         // of the tokens with a bias
  const int b = blockIdx.y, t = threadIdx.x;
  const T* x = static_cast<const T*>(p.logits) + (size_t)b * p.ld;
  float* y = p.out + (size_t)b * p.ldo;
  const int off = (int)(((uintptr_t)y >> 2) & 3);                       // tokens past a boundary at the row's start
  const bool wide = ((uintptr_t)y & 3) == 0 && ((uintptr_t)x / sizeof(T) & 3) == (unsigned)off;
  const int lo = (int)blockIdx.x * SLICE - (wide ? off : 0);            // (the first slice starts up to three tokens in front of the row)
  const bool history = p.tokens != nullptr;
  const bool table = history || p.n_bias;
#pragma unroll
  for (int k = 0; k < N; ++k) if (table) reinterpret_cast<uint4*>(lr_count)[k * TH + t] = make_uint4(0, 0, 0, 0);
  pdl_wait();
  pdl_launch_dependents();
  // ---- all that is read, on its way together
  const int len = p.lengths ? min(p.lengths[p.lengths_n > 1 ? b : 0], p.T) : p.T;
  const int start = p.starts ? max(p.starts[p.starts_n > 1 ? b : 0], 0) : 0;
  const int prompt = p.prompts ? p.prompts[p.prompts_n > 1 ? b : 0] : 0;
  const float r = p.rep ? p.rep[b] : p.rep1, f = p.freq ? p.freq[b] : p.freq1, pr = p.pres ? p.pres[b] : p.pres1;
  // v / r as v (1 / r) in 64 bits, rounded once to 32, over the whole range of r.  It is v / r rounded: with v = m 2^i, r = n 2^j (m, n < 2^24 whole) a midpoint M 2^l of two fp32
  // numbers (M < 2^25, odd) is v / r only if M divides m, which is smaller; otherwise |m 2^.. - M n 2^..| >= 1 keeps v / r 2^-49 of its size away, and the two roundings
  // in 64 bits are 2^-52 together.  (Below 2^-126 midpoints are shorter, and the last bit may be the other one.)  us of the calls above, 1, 17, 96 rows, on one box: a division in fp32
  // 2.55, 5.9, 30.1; this 2.24, 5.45, 29.7.
  const double inv_r = 1.0 / (double)r;
  const int* row = p.tokens + (size_t)b * p.ldt;
  // history: AHEAD groups of four tokens per thread before its length is known, each on a 16-byte boundary (the first up to three tokens in front of the row)
  constexpr int AHEAD = 2;
  const int past = (int)(((uintptr_t)row >> 2) & 3);
  const int limit = history ? p.T : 0;
  auto group = [&](int i, int end) {
    if (i >= 0 && i + 4 <= end) return *reinterpret_cast<const int4*>(row + i);
    int4 a = make_int4(-1, -1, -1, -1);
    if (i >= end) return a;
    a.x = i >= 0 && i < end ? row[i] : -1;
    a.y = i + 1 >= 0 && i + 1 < end ? row[i + 1] : -1;
    a.z = i + 2 >= 0 && i + 2 < end ? row[i + 2] : -1;
    a.w = i + 3 < end ? row[i + 3] : -1;                                // (never in front of the row)
    return a;
  };
  int4 said[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) said[u] = group(4 * (u * TH + t) - past, limit);
  const int* ids = p.bias_ids + (size_t)b * p.ldb;
  const float* bias = p.bias + (size_t)b * p.ldb;
  const int id0 = t < p.n_bias ? ids[t] : -1, id1 = t + TH < p.n_bias ? ids[t + TH] : -1;
  const float bias0 = t < p.n_bias ? bias[t] : 0.f, bias1 = t + TH < p.n_bias ? bias[t + TH] : 0.f;
  float v[N][4];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = lo + 4 * (k * TH + t);
    if (wide && i >= 0 && i + 4 <= p.V) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(x + i);
        v[k][0] = a.x; v[k][1] = a.y; v[k][2] = a.z; v[k][3] = a.w;
      } else {
        T a[4];
        *reinterpret_cast<uint2*>(a) = *reinterpret_cast<const uint2*>(x + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = (float)a[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = i + e >= 0 && i + e < p.V ? (float)x[i + e] : 0.f;
    }
  }
  unsigned word[N], next[N];                                            // the mask's word with a group's first token, and the one behind it where the group ends there
  const int words = (p.V + 31) >> 5;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = lo + 4 * (k * TH + t), w = i >> 5;                    // (-1 in front of the row)
    word[k] = next[k] = ~0u;
    if (p.allowed) {
      const unsigned* mask = p.allowed + (size_t)b * p.lda;
      if (w >= 0 && w < words) word[k] = __ldg(mask + w);
      if (off && (i & 31) > 28 && w + 1 < words) next[k] = __ldg(mask + w + 1);
    }
  }
  __syncthreads();
  if (history) {
    // (ids outside the vocabulary: beyond the slice, or words of it that stand for no token)
    const unsigned span = (unsigned)max(len - start, 0);
    auto count = [&](int i, int id) {
      const unsigned at = (unsigned)id - (unsigned)lo;
      if (at < (unsigned)SLICE && (unsigned)(i - start) < span) {
        if (i < prompt) atomicOr(&lr_count[at], LR_SAID);
        else atomicAdd(&lr_count[at], 1u);
      }
    };
    auto count4 = [&](int i, int4 a) {                                  // (few groups have a token of the slice)
      if (min(min((unsigned)(a.x - lo), (unsigned)(a.y - lo)), min((unsigned)(a.z - lo), (unsigned)(a.w - lo))) >= (unsigned)SLICE) return;
      count(i, a.x); count(i + 1, a.y); count(i + 2, a.z); count(i + 3, a.w);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) count4(4 * (u * TH + t) - past, said[u]);
    for (int i0 = 4 * (AHEAD * TH + t) - past; i0 < len; i0 += 4 * AHEAD * TH) {        // AHEAD loads in flight
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) said[u] = group(i0 + 4 * u * TH, len);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) count4(i0 + 4 * u * TH, said[u]);
    }
  }
  // ---- biases: whoever marks a token first leaves the value, the others say that there are more: then it is the sum
  unsigned mine = 0;                                                    // bit k: this thread was first with entry t + k TH
  for (int i = t, k = 0; i < p.n_bias; i += TH, ++k) {
    const int id = k == 0 ? id0 : (k == 1 ? id1 : ids[i]);
    const unsigned at = (unsigned)id - (unsigned)lo;
    if (at < (unsigned)SLICE && id >= 0 && id < p.V) {
      if (atomicOr(&lr_count[at], LR_BIAS) & LR_BIAS) atomicOr(&lr_count[at], LR_MORE);
      else { lr_value[at] = k == 0 ? bias0 : (k == 1 ? bias1 : bias[i]); mine |= 1u << k; }
    }
  }
  if (p.n_bias) {
    __syncthreads();
    for (unsigned left = mine; left; left &= left - 1) {
      const int id = ids[t + (__ffs(left) - 1) * TH];
      if (!(lr_count[id - lo] & LR_MORE)) continue;
      float sum = 0.f;
      for (int j = 0; j < p.n_bias; ++j) if (ids[j] == id) sum += bias[j];
      lr_value[id - lo] = sum;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = lo + 4 * (k * TH + t);
    const unsigned bits = __funnelshift_r(word[k], next[k], i & 31);
    if (table) {
      const uint4 c4 = reinterpret_cast<const uint4*>(lr_count)[k * TH + t];
      const unsigned c[4] = {c4.x, c4.y, c4.z, c4.w};
      if (c4.x | c4.y | c4.z | c4.w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned n = c[e] & LR_COUNT;
          const float quo = (float)((double)v[k][e] * inv_r), pen = v[k][e] > 0.f ? quo : v[k][e] * r;
          if (c[e] & (LR_COUNT | LR_SAID)) v[k][e] = pen;
          if (n) v[k][e] = v[k][e] - f * (float)n - pr;
          if (c[e] & LR_BIAS) v[k][e] += lr_value[4 * (k * TH + t) + e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) if (!((bits >> e) & 1u)) v[k][e] = -INFINITY;
    if (wide && i >= 0 && i + 4 <= p.V) {
      *reinterpret_cast<float4*>(y + i) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) if (i + e >= 0 && i + e < p.V) y[i + e] = v[k][e];
    }
  }
}

template <typename T, int TH, int N>
static cudaError_t lr_launch(const RulesParams& p, int B, cudaStream_t st) {
  constexpr int SLICE = 4 * N * TH;
  const size_t smem = (size_t)SLICE * 4 * (p.n_bias ? 2 : (p.tokens ? 1 : 0));
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(logit_rules_kernel<T, TH, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(logit_rules_kernel<T, TH, N>, dim3((p.V + 3 + SLICE - 1) / SLICE, B), dim3(TH), smem, st, p);
}
template <typename T>
static cudaError_t lr_dispatch(const RulesParams& p, int B, cudaStream_t st) {
  // Few rows: the smallest slices, for more SMs; many: large ones, because every slice's CTA walks the row's whole history.  us in a graph on one B200, 17 x 128259
  // with 2049 tokens of history and 96 x 128256 with 4000: four groups for each of 128, 256, 512 threads 6.0, 5.8, 5.4 and 38, 32, 30; two for 512 7.4 and 40.
  const long groups = ((long)p.V + 3) / 4 * B / 256;                   // CTAs of 256 threads with one group each
  if (groups <= 2 * 148) return lr_launch<T, 256, 1>(p, B, st);
  if (groups <= 6 * 148) return lr_launch<T, 256, 2>(p, B, st);
  return lr_launch<T, 512, 4>(p, B, st);
}

}  // namespace jl

using namespace jl;

extern "C" JL_API int jl_logit_rules(const void* logits, int dtype, int B, int V, int ld, float* out, int ldo, const int* tokens, int T, int ldt, const int* starts,
                                     int starts_n, const int* lengths, int lengths_n, const int* prompts, int prompts_n, const float* rep, float rep1,
                                     const float* freq, float freq1, const float* pres, float pres1, const int* bias_ids, const float* bias, int n_bias, int ldb,
                                     const void* allowed, int lda, void* stream) {
  if (B == 0 || V == 0) return JL_OK;
  JL_CHECK_ARG(logits && out && B > 0 && V > 0 && B <= 65535 && (ld >= V || ld == 0) && ldo >= V, "jl_logit_rules: %d rows of %d logits, pitches %d and %d", B, V, ld, ldo);
  JL_CHECK_ARG(V <= (1 << 30) && (uintptr_t)logits % (dtype == 0 ? 4 : 2) == 0 && (uintptr_t)out % 4 == 0, "jl_logit_rules: vocabulary of %d, or misplaced logits", V);
  JL_CHECK_ARG(dtype >= 0 && dtype <= 2, "jl_logit_rules: dtype %d (0 fp32, 1 bf16, 2 fp16)", dtype);
  JL_CHECK_ARG(tokens == nullptr || (T >= 0 && ldt >= T), "jl_logit_rules: history of %d tokens, pitch %d", T, ldt);
  for (int n : {starts ? starts_n : 1, lengths ? lengths_n : 1, prompts ? prompts_n : 1})
    JL_CHECK_ARG(n == 1 || n == B, "jl_logit_rules: %d row bounds for %d rows", n, B);
  JL_CHECK_ARG(n_bias >= 0 && n_bias <= 8192 && (n_bias == 0 || (bias_ids && bias && (ldb == 0 || ldb >= n_bias))), "jl_logit_rules: %d biases, pitch %d", n_bias, ldb);
  JL_CHECK_ARG(allowed == nullptr || lda == 0 || lda >= (V + 31) / 32, "jl_logit_rules: mask rows of %d words for %d tokens", lda, V);
  RulesParams p{};
  p.logits = logits; p.ld = ld; p.out = out; p.ldo = ldo; p.V = V;
  p.tokens = T > 0 ? tokens : nullptr; p.ldt = ldt; p.T = T;
  p.starts = starts; p.starts_n = starts_n; p.lengths = lengths; p.lengths_n = lengths_n; p.prompts = prompts; p.prompts_n = prompts_n;
  p.rep = rep; p.rep1 = rep1; p.freq = freq; p.freq1 = freq1; p.pres = pres; p.pres1 = pres1;
  p.bias_ids = bias_ids; p.bias = bias; p.n_bias = n_bias; p.ldb = ldb;
  p.allowed = (const unsigned*)allowed; p.lda = lda;
  cudaError_t e = dtype == 0 ? lr_dispatch<float>(p, B, (cudaStream_t)stream)
                             : (dtype == 1 ? lr_dispatch<__nv_bfloat16>(p, B, (cudaStream_t)stream) : lr_dispatch<__half>(p, B, (cudaStream_t)stream));
  JL_CUDA(e);
  return JL_OK;
}
