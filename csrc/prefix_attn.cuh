// Attention over keys that the rows of a group share and over every row's own keys: what prefix_attn.cu (tcgen05 tiles) and the one-token kernel of
// decode_attn_fused.cu (the own keys, and the join) agree on.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace jl {

// Partial results of the shared keys: per (token, head) `splits` triples, o (sum of weights times values, fp32 [hd]) and (m, l): the reference exponent in
// base 2 and the sum of weights against it.  A split without keys has l = 0 and no o.
struct PrefixParts {
  const float* o;                   // [tokens * nh][splits][hd]
  const float2* ml;                 // [tokens * nh][splits]
  int splits;
};

// One new token of every row: rotation and append of its key, attention over the row's own keys, joined with the partial results of the shared ones.
struct PrefixStep {
  const __nv_bfloat16* qkv;         // [B, (nh + 2 nkv) hd], not rotated
  __nv_bfloat16* k_cache;           // [B][nkv][T][hd]
  __nv_bfloat16* v_cache;
  const float* cos_t;               // [max_pos, hd / 2]
  const float* sin_t;
  const int* cache_len;
  const int* pad_left;              // [B] or nullptr
  const int* prefix_len;            // [groups] or nullptr: all P slots
  const int* prefix_pad;            // [groups] or nullptr
  __nv_bfloat16* out;               // [B, nh hd]
  void* scratch;                    // of the own keys' splits
  int B, rows, nh, nkv, hd, P, T, max_pos;
  float scale;
  PrefixParts parts;
};

size_t prefix_step_scratch_bytes(int B, int nh, int nkv, int hd);
int prefix_step_launch(const PrefixStep& s, cudaStream_t st);

}  // namespace jl
