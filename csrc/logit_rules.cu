// The rules of a request on the logits of a step: penalties for tokens that occurred, biases, a mask of allowed tokens.
//
//   x = logits[b, v]
//   v occurs in tokens[b, start_b .. len_b):               x = x > 0 ? x / r_b : x r_b                    (repetition)
//   n = occurrences in tokens[b, prompt_b .. len_b), n > 0: x = x - f_b n - p_b                           (frequency, presence)
//   every entry i with bias_ids[b, i] == v:                x = x + bias[b, i]                             (in the order of the entries)
//   bit v of allowed[b] is zero:                           x = -infinity
//
// A CTA owns a slice of one row's vocabulary and keeps, per token of the slice, a count in shared memory: bit 31 = occurred, the rest = occurrences behind the
// prompt (whole numbers: the order of the atomics does not show), and beside it the sum of the biases when there are any.  It walks the row's
// history, counts what falls into its slice, then passes over the slice once.  No state is kept between calls: the history is the sequence
// buffer that the decode loop writes anyway, so forks, restarts and replayed graphs need nothing.
#include "common.cuh"
#include "jllama_b200.h"

#include <cuda_fp16.h>

namespace jl {

constexpr int LR_THREADS = 512;

struct RulesParams {
  const void* logits; int ld;
  float* out; int ldo;
  int V, slice;
  const int* tokens; int ldt, T;
  const int* starts; int starts_n;                  // [B] or one for all rows (n = 1), or nullptr
  const int* lengths; int lengths_n;
  const int* prompts; int prompts_n;
  const float* rep; const float* freq; const float* pres;       // [B] or nullptr: the scalar
  float rep1, freq1, pres1;
  const int* bias_ids; const float* bias; int n_bias, ldb;
  const unsigned* allowed; int lda;
};

template <typename T> __device__ __forceinline__ float lr_load(const T* p) { return (float)*p; }

template <typename T>
__global__ void __launch_bounds__(LR_THREADS) logit_rules_kernel(const RulesParams p) {
  extern __shared__ unsigned lr_count[];
  float* s_bias = reinterpret_cast<float*>(lr_count + p.slice);
  const int b = blockIdx.y, lo = blockIdx.x * p.slice, n = min(p.slice, p.V - lo);
  const bool history = p.tokens != nullptr;
  if (history)
    for (int i = threadIdx.x; i < n; i += LR_THREADS) lr_count[i] = 0;
  if (p.n_bias)
    for (int i = threadIdx.x; i < n; i += LR_THREADS) s_bias[i] = 0.f;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  if (history) {
    const int len = p.lengths ? min(p.lengths[p.lengths_n > 1 ? b : 0], p.T) : p.T;
    const int start = p.starts ? max(p.starts[p.starts_n > 1 ? b : 0], 0) : 0;
    const int prompt = p.prompts ? p.prompts[p.prompts_n > 1 ? b : 0] : 0;
    const int* row = p.tokens + (size_t)b * p.ldt;
    for (int i = start + threadIdx.x; i < len; i += LR_THREADS) {
      const unsigned v = (unsigned)row[i] - (unsigned)lo;
      if (v < (unsigned)n) {
        if (i < prompt) atomicOr(&lr_count[v], 0x80000000u);
        else atomicAdd(&lr_count[v], 1u);
      }
    }
  }
  if (p.n_bias && threadIdx.x < 32) {
    // one warp, the entries in order: those of a token that stand in one load are added one after the other
    const int* ids = p.bias_ids + (size_t)b * p.ldb;
    const float* val = p.bias + (size_t)b * p.ldb;
    for (int i0 = 0; i0 < p.n_bias; i0 += 32) {
      const int i = i0 + (int)threadIdx.x;
      const int id = i < p.n_bias ? (int)((unsigned)ids[i] - (unsigned)lo) : -1;
      const float x = i < p.n_bias ? val[i] : 0.f;
      const bool mine = (unsigned)id < (unsigned)n;
      const unsigned same = __match_any_sync(0xffffffffu, mine ? id : -1 - (int)threadIdx.x);
      const int before = __popc(same & ((1u << threadIdx.x) - 1u));
      int most = mine ? __popc(same) : 0;
      most = __reduce_max_sync(0xffffffffu, most);
      for (int k = 0; k < most; ++k) {
        if (mine && before == k) s_bias[id] += x;
        __syncwarp();
      }
    }
  }
  __syncthreads();
  const float r = p.rep ? p.rep[b] : p.rep1, f = p.freq ? p.freq[b] : p.freq1, pr = p.pres ? p.pres[b] : p.pres1;
  const T* x = static_cast<const T*>(p.logits) + (size_t)b * p.ld + lo;
  float* y = p.out + (size_t)b * p.ldo + lo;
  const unsigned* bits = p.allowed ? p.allowed + (size_t)b * p.lda : nullptr;
  for (int i = threadIdx.x; i < n; i += LR_THREADS) {
    float v = lr_load(x + i);
    if (history) {
      const unsigned c = lr_count[i];
      if (c) {
        v = v > 0.f ? __fdiv_rn(v, r) : v * r;
        const unsigned k = c & 0x7fffffffu;
        if (k) v = v - f * (float)k - pr;
      }
    }
    if (p.n_bias) v += s_bias[i];
    if (bits && !((bits[(lo + i) >> 5] >> ((lo + i) & 31)) & 1u)) v = -INFINITY;
    y[i] = v;
  }
}

}  // namespace jl

using namespace jl;

extern "C" JL_API int jl_logit_rules(const void* logits, int dtype, int B, int V, int ld, float* out, int ldo, const int* tokens, int T, int ldt, const int* starts,
                                     int starts_n, const int* lengths, int lengths_n, const int* prompts, int prompts_n, const float* rep, float rep1,
                                     const float* freq, float freq1, const float* pres, float pres1, const int* bias_ids, const float* bias, int n_bias, int ldb,
                                     const void* allowed, int lda, void* stream) {
  if (B == 0 || V == 0) return JL_OK;
  JL_CHECK_ARG(logits && out && B > 0 && V > 0 && B <= 65535 && ld >= V && ldo >= V, "jl_logit_rules: %d rows of %d logits, pitches %d and %d", B, V, ld, ldo);
  JL_CHECK_ARG(dtype >= 0 && dtype <= 2, "jl_logit_rules: dtype %d (0 fp32, 1 bf16, 2 fp16)", dtype);
  JL_CHECK_ARG(tokens == nullptr || (T >= 0 && ldt >= T), "jl_logit_rules: history of %d tokens, pitch %d", T, ldt);
  for (int n : {starts ? starts_n : 1, lengths ? lengths_n : 1, prompts ? prompts_n : 1})
    JL_CHECK_ARG(n == 1 || n == B, "jl_logit_rules: %d row bounds for %d rows", n, B);
  JL_CHECK_ARG(n_bias >= 0 && (n_bias == 0 || (bias_ids && bias && (ldb == 0 || ldb >= n_bias))), "jl_logit_rules: %d biases, pitch %d", n_bias, ldb);
  JL_CHECK_ARG(allowed == nullptr || lda == 0 || lda >= (V + 31) / 32, "jl_logit_rules: mask rows of %d words for %d tokens", lda, V);
  RulesParams p{};
  p.logits = logits; p.ld = ld; p.out = out; p.ldo = ldo; p.V = V;
  p.tokens = T > 0 ? tokens : nullptr; p.ldt = ldt; p.T = T;
  p.starts = starts; p.starts_n = starts_n; p.lengths = lengths; p.lengths_n = lengths_n; p.prompts = prompts; p.prompts_n = prompts_n;
  p.rep = rep; p.rep1 = rep1; p.freq = freq; p.freq1 = freq1; p.pres = pres; p.pres1 = pres1;
  p.bias_ids = bias_ids; p.bias = bias; p.n_bias = n_bias; p.ldb = ldb;
  p.allowed = (const unsigned*)allowed; p.lda = lda;
  p.slice = 4096;
  const dim3 grid((V + p.slice - 1) / p.slice, B);
  const size_t smem = (size_t)p.slice * 4 * (n_bias ? 2 : 1);
  cudaError_t e;
  if (dtype == 0) e = launch_pdl(logit_rules_kernel<float>, grid, dim3(LR_THREADS), smem, (cudaStream_t)stream, p);
  else if (dtype == 1) e = launch_pdl(logit_rules_kernel<__nv_bfloat16>, grid, dim3(LR_THREADS), smem, (cudaStream_t)stream, p);
  else e = launch_pdl(logit_rules_kernel<__half>, grid, dim3(LR_THREADS), smem, (cudaStream_t)stream, p);
  JL_CUDA(e);
  return JL_OK;
}
