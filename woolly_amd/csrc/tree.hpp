// tree.hpp -- launchers of the operators that verify a tree of drafted tokens
// (tree_attention.hip, tree.hip, logits.hip).  Arguments have been checked by
// the C entry points; the launchers choose kernels and launch them.
#pragma once

#include "wh_common.hpp"

namespace wh {

// Nodes of one tree, and sequences of one call, that the kernels take.
constexpr size_t kMaxTreeNodes = WH_MAX_TREE_NODES;
constexpr size_t kMaxTreeSeqs = 1024;

struct TreeAttnArgs {
  const float* q;           // [n_seqs * n_tree] rows of ldq elements
  const float* k;           // rows of ldkv elements
  const float* v;
  size_t ldq, ldkv;
  const int32_t* parents;   // [n_seqs][n_tree]
  const uint32_t* ctx_len;  // [n_seqs]
  size_t n_seqs, n_tree;
  void* k_cache;            // f16 [n_seqs][max_ctx][n_kv_heads][head_dim]
  void* v_cache;
  size_t max_ctx, n_heads, n_kv_heads, head_dim;
  const float* inv_freq;
  float* out;               // [n_seqs * n_tree][n_heads * head_dim]
};
bool tree_attention_shape_ok(size_t n_heads, size_t n_kv_heads, size_t head_dim);
size_t tree_attention_workspace_bytes(size_t n_seqs, size_t n_tree, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                      size_t max_ctx);
int launch_tree_attention(const TreeAttnArgs& a, void* workspace, hipStream_t stream);

}  // namespace wh

namespace whd {

// Ancestors of every node of one tree in LDS, by pointer doubling: bit a of
// mask[t] is set where a is t itself or an ancestor of t; depth[t] counts the
// ancestors.  A node whose parent is neither -1 nor an earlier node is absent,
// and so are all below it: their masks are 0.  Every thread of the workgroup
// calls it (thread i < 128 keeps node i); 7 rounds join 2^7 = 128 levels.
struct TreeScratch {
  uint32_t mask[2][128][4];
  int jump[2][128];
};
__device__ __forceinline__ const uint32_t (*tree_ancestors(const int32_t* __restrict__ parents, int n_tree,
                                                           TreeScratch& ts))[4] {
  constexpr int kCache = -1, kAbsent = -2;
  const int t = threadIdx.x;
  if (t < 128) {
    int p = kAbsent;
    if (t < n_tree) {
      const int g = parents[t];
      p = g == -1 ? kCache : (g >= 0 && g < t ? g : kAbsent);
    }
    for (int w = 0; w < 4; w++) ts.mask[0][t][w] = (t >> 5) == w ? 1u << (t & 31) : 0u;
    ts.jump[0][t] = p;
  }
  int cur = 0;
  for (int round = 0; round < 7; round++) {
    __syncthreads();
    if (t < 128) {
      const int j = ts.jump[cur][t];
      uint32_t m[4];
      for (int w = 0; w < 4; w++) m[w] = ts.mask[cur][t][w] | (j >= 0 ? ts.mask[cur][j][w] : 0u);
      for (int w = 0; w < 4; w++) ts.mask[cur ^ 1][t][w] = m[w];
      ts.jump[cur ^ 1][t] = j >= 0 ? ts.jump[cur][j] : j;
    }
    cur ^= 1;
  }
  __syncthreads();
  if (t < 128 && ts.jump[cur][t] != kCache) {
    for (int w = 0; w < 4; w++) ts.mask[cur][t][w] = 0u;
  }
  __syncthreads();
  return ts.mask[cur];
}

}  // namespace whd
