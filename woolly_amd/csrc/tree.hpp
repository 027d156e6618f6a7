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

// Largest float (NaN passed over) and smallest number over the wave's 64 lanes, in
// every lane: swaps within rows of 16 lanes (DPP), then of rows and halves
// (v_permlane16_swap, v_permlane32_swap).  No LDS round trips, as __shfl_xor
// would take: some 60 cycles instead of 700.
template <typename Op>
__device__ __forceinline__ uint32_t wave_join(uint32_t v, Op op) {
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xF, 0xF, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xF, 0xF, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xF, 0xF, false)));
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x140, 0xF, 0xF, false)));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = op(static_cast<uint32_t>(a[0]), static_cast<uint32_t>(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return op(static_cast<uint32_t>(b[0]), static_cast<uint32_t>(b[1]));
}
__device__ __forceinline__ float wave_max(float v) {
  return __builtin_bit_cast(float, wave_join(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
  }));
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  return wave_join(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// A barrier for what goes through LDS only: __syncthreads() would also wait for
// the global loads and stores in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The path from the cache to node t of one tree: bit a is set where a is t itself
// or an ancestor of t; depth counts its ancestors.  A node whose parent is
// neither -1 nor an earlier node is absent, and so are all below it: no bits.
// One wave walks by itself, without LDS or barriers: its lanes hold the parents
// and every step reads one of them as a scalar (some 20 cycles; a path has as
// many steps as nodes, at most 128).
struct TreePath {
  unsigned long long lo, hi;  // nodes 0..63, 64..127
  int depth;
  __device__ __forceinline__ bool present() const { return (lo | hi) != 0; }
  __device__ __forceinline__ bool has(int a) const { return ((a < 64 ? lo : hi) >> (a & 63)) & 1u; }
};
// A tree's parents over the lanes of a wave (lane l: nodes l and l + 64); one
// that is no earlier node, but not -1 either, is -2.
struct TreeLanes {
  int p0, p1;
};
__device__ __forceinline__ TreeLanes tree_lanes(const int32_t* __restrict__ parents, int n_tree) {
  const int lane = threadIdx.x & 63;
  const int a = lane < n_tree ? parents[lane] : -2, b = lane + 64 < n_tree ? parents[lane + 64] : -2;
  return TreeLanes{a >= lane ? -2 : a, b >= lane + 64 ? -2 : b};
}
// Cache rows that a tree takes: up to its last node whose parent is -1 or an earlier one.
__device__ __forceinline__ uint32_t tree_rows(const TreeLanes& tree) {
  const unsigned long long lo = __ballot(tree.p0 >= -1), hi = __ballot(tree.p1 >= -1);
  return hi ? 128 - __builtin_clzll(hi) : lo ? 64 - __builtin_clzll(lo) : 0;
}
__device__ __forceinline__ TreePath tree_path(const TreeLanes& tree, int t) {
  TreePath p{0, 0, -1};
  int at = t;
  while (at >= 0) {  // falls with every step
    if (at < 64) p.lo |= 1ull << at; else p.hi |= 1ull << (at - 64);
    p.depth++;
    const int a = __builtin_amdgcn_readlane(tree.p0, at & 63), b = __builtin_amdgcn_readlane(tree.p1, at & 63);
    at = at < 64 ? a : b;
  }
  if (at != -1) p = TreePath{0, 0, 0};
  return p;
}

}  // namespace whd
