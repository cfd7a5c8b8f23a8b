// Partial results of attention over parts of a key range: for each part, kv head and query row the running
// maximum m (in units of log 2) and the sum l = sum exp2(s - m), and the weighted sum O = sum exp2(s - m) v,
// all in 32 bits. A part that saw no key has l = 0.
#pragma once
#include "common.cuh"

namespace {

struct AttnParts {
  float* o;                  // [splits][nkv][rows][128]
  float2* ml;                // [splits][nkv][rows]
  const int32_t* keys;       // null: every split is written; else as many as `keys` has tiles of `tile` keys
  int splits, nkv, rows, tile;
  __device__ __forceinline__ size_t row(int split, int kh, size_t r) const {
    return ((size_t)split * nkv + kh) * rows + r;
  }
};

#ifdef __CUDACC__
// Splits that hold results: a range of few tiles leaves the others out.
__device__ __forceinline__ int parts_used(const AttnParts& p) {
  if (p.keys == nullptr) return p.splits;
  const int n = max(0, __ldcg(p.keys));
  return min(p.splits, n / p.tile + (n % p.tile != 0));
}
#endif

}  // namespace

// Rows over one range of keys that all of them see (a shared prefix), as partial results on the prompt
// attention's kernel: q [tokens][n_q_heads][128] against keys [0, *d_len) of a one-sequence cache.
int q_attention_parts_tc(const void* d_q, const q_kv_layout_t* kv, const int32_t* d_len, float* parts_o,
                         float* parts_ml, int splits, int tokens, int n_q_heads, float scale, void* stream);
