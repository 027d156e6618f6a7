// tree.hip -- what follows the verification of a tree of drafted tokens: the
// walk along the chosen tokens, and the accepted rows moved together in the KV
// caches of every layer.
//
// Neither moves enough to be bound by memory: a walk reads 1.5 KB at most and a
// step keeps a few rows of each layer.  Both are one launch whose latency is
// that of its dependent loads: 2.3 us for one walk over 26 nodes, 3.8 for 256
// over 64; 4.1 us for 7 rows in 32 layers, 4.2 for 16 sequences in 24.
#include <algorithm>
#include <memory>
#include <new>

#include "tree.hpp"

namespace {

constexpr uint32_t kNoToken = 0xFFFFFFFFu;

struct AcceptParams {
  const uint32_t* tokens;   // [n_seqs][n_tree]
  const int32_t* parents;
  const uint32_t* picked;
  uint32_t* path;
  uint32_t* n_accepted;
  uint32_t* next_token;
  const uint32_t* ctx_len;
  uint32_t* ctx_len_out;
  uint32_t* history;
  size_t history_stride;
  uint32_t n_tree;
  uint32_t max_ctx;         // cache rows that hold the trees, 0: whatever
};

// One wave per sequence, lane l holding nodes l and l + 64.  From node 0 the
// walk goes to the first child that carries the token picked at the node; all
// children are compared at once.  A tree that its cache did not hold (by tree_rows'
// measure) has nothing accepted: no row of it is there to keep.
__global__ __launch_bounds__(64) void tree_accept_kernel(const AcceptParams P) {
  const uint32_t s = blockIdx.x, lane = threadIdx.x;
  const size_t row = static_cast<size_t>(s) * P.n_tree;
  int32_t parent[2];
  uint32_t token[2], picked[2], order[2] = {kNoToken, kNoToken};
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const uint32_t t = lane + 64 * u;
    const bool in = t < P.n_tree;
    parent[u] = in ? P.parents[row + t] : -2;
    token[u] = in ? P.tokens[row + t] : 0u;
    picked[u] = in ? P.picked[row + t] : kNoToken;
  }
  const uint32_t ctx = P.ctx_len ? P.ctx_len[s] : 0;
  uint32_t n = 0, next = kNoToken;
  int at = __shfl(parent[0], 0, 64) == -1 ? 0 : -1;
  if (P.max_ctx) {
    const uint32_t rows = whd::tree_rows(whd::TreeLanes{parent[0] >= static_cast<int>(lane) ? -2 : parent[0],
                                                        parent[1] >= static_cast<int>(lane) + 64 ? -2 : parent[1]});
    if (ctx > P.max_ctx || rows > P.max_ctx - ctx) at = -1;
  }
  while (at >= 0) {  // at grows with every step: at most n_tree steps
    if (lane == static_cast<uint32_t>(at & 63)) order[at >> 6] = n;
    n++;
    const uint32_t a = __shfl(picked[0], at & 63, 64), b = __shfl(picked[1], at & 63, 64);
    next = at < 64 ? a : b;
    // a child comes behind its parent, anything else is not there
    const bool c0 = parent[0] == at && static_cast<int>(lane) > at && token[0] == next && next != kNoToken;
    const bool c1 = parent[1] == at && static_cast<int>(lane) + 64 > at && token[1] == next && next != kNoToken;
    const unsigned long long m0 = __ballot(c0), m1 = __ballot(c1);
    at = m0 ? __builtin_ctzll(m0) : m1 ? 64 + __builtin_ctzll(m1) : -1;
  }
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const uint32_t t = lane + 64 * u;
    if (t < P.n_tree && t >= n) P.path[row + t] = kNoToken;
    if (order[u] == kNoToken) continue;
    P.path[row + order[u]] = t;
    const size_t p = static_cast<size_t>(ctx) + order[u];
    if (P.history && p < P.history_stride) P.history[s * P.history_stride + p] = token[u];
  }
  if (lane == 0) {
    P.n_accepted[s] = n;
    P.next_token[s] = next;
    if (P.ctx_len_out) P.ctx_len_out[s] = ctx + n;
  }
}

// Layers of one launch: their cache pointers are kernel arguments.
constexpr int kCompactLayers = 64;
constexpr int kCompactBatch = 8;
typedef uint32_t piece16 __attribute__((ext_vector_type(4)));  // arrays of HIP's uint4 end up in scratch memory here
struct CompactParams {
  piece16* cache[2 * kCompactLayers];
  const uint32_t* path;
  const uint32_t* n_accepted;
  const uint32_t* ctx_len;
  size_t max_ctx;
  uint32_t row16;  // 16-byte pieces per cache row
  uint32_t n_tree;
};

// grid: (2 * layers, n_seqs, pieces / 256).  A thread moves one 16-byte column
// of the accepted rows: 8 rows are loaded before the first is stored.  Row i
// comes from path[i] >= i (paths ascend), so a row is read before the same
// thread stores over it, and no other thread touches its column.
__global__ __launch_bounds__(256) void kv_compact_kernel(const CompactParams P) {
  const uint32_t s = blockIdx.y, c = blockIdx.z * 256 + threadIdx.x;
  const uint32_t n = P.n_accepted[s], after = P.ctx_len[s];
  if (n > P.n_tree || n > after || after > P.max_ctx) return;
  const uint32_t first = after - n;
  if (c >= P.row16) return;
  piece16* base = P.cache[blockIdx.x] + (static_cast<size_t>(s) * P.max_ctx + first) * P.row16 + c;
  const uint32_t* path = P.path + static_cast<size_t>(s) * P.n_tree;
  for (uint32_t i0 = 0; i0 < n; i0 += kCompactBatch) {
    piece16 v[kCompactBatch];
    bool moved[kCompactBatch];
#pragma unroll
    for (int j = 0; j < kCompactBatch; j++) {
      const uint32_t i = i0 + j;
      const uint32_t p = i < n ? path[i] : 0;
      // a row that stays, or that the cache does not hold, is not moved: its load takes row 0
      moved[j] = p > i && p < P.n_tree && static_cast<size_t>(first) + p < P.max_ctx;
      v[j] = base[static_cast<size_t>(moved[j] ? p : 0) * P.row16];
    }
#pragma unroll
    for (int j = 0; j < kCompactBatch; j++)
      if (moved[j]) base[static_cast<size_t>(i0 + j) * P.row16] = v[j];
  }
}

}  // namespace

// max_ctx 0: the caches are not looked at.
static int accept(const uint32_t* tokens, const int32_t* parents, const uint32_t* picked, size_t n_seqs, size_t n_tree,
                  uint32_t* path, uint32_t* n_accepted, uint32_t* next_token, const uint32_t* ctx_len,
                  uint32_t* ctx_len_out, uint32_t* history, size_t history_stride, size_t max_ctx, wh_stream_t stream) {
  // a launch has less than 2^32 threads, 64 of them to a sequence
  if (n_tree > wh::kMaxTreeNodes || n_seqs >> 26)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "tree_accept: %zu nodes (at most %zu) of %zu sequences (less than 2^26)", n_tree,
                         wh::kMaxTreeNodes, n_seqs);
  if (n_seqs == 0 || n_tree == 0) return WH_OK;
  if (!tokens || !parents || !picked || !path || !n_accepted || !next_token)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "tree_accept: null pointer");
  if ((ctx_len_out || history || max_ctx) && !ctx_len)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "tree_accept: ctx_len_out, history and max_ctx need ctx_len");
  const void* ptrs[] = {tokens, parents, picked, path, n_accepted, next_token, ctx_len, ctx_len_out, history};
  for (const void* p : ptrs)
    if (!wh::aligned(p, 4)) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "tree_accept: arrays must be 4-byte aligned");
  const AcceptParams P{tokens,  parents,     picked,  path,           n_accepted, next_token,
                       ctx_len, ctx_len_out, history, history_stride, static_cast<uint32_t>(n_tree),
                       static_cast<uint32_t>(max_ctx)};
  tree_accept_kernel<<<static_cast<unsigned>(n_seqs), 64, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
  WH_LAUNCH_CHECK("tree accept launch");
  return WH_OK;
}

WH_API int wh_tree_accept(const uint32_t* tokens, const int32_t* parents, const uint32_t* picked, size_t n_seqs,
                          size_t n_tree, uint32_t* path, uint32_t* n_accepted, uint32_t* next_token,
                          const uint32_t* ctx_len, uint32_t* ctx_len_out, uint32_t* history, size_t history_stride,
                          wh_stream_t stream) {
  return accept(tokens, parents, picked, n_seqs, n_tree, path, n_accepted, next_token, ctx_len, ctx_len_out, history,
                history_stride, 0, stream);
}

WH_API int wh_tree_accept_in_cache(const uint32_t* tokens, const int32_t* parents, const uint32_t* picked, size_t n_seqs,
                                   size_t n_tree, uint32_t* path, uint32_t* n_accepted, uint32_t* next_token,
                                   const uint32_t* ctx_len, uint32_t* ctx_len_out, uint32_t* history,
                                   size_t history_stride, size_t max_ctx, wh_stream_t stream) {
  if (max_ctx == 0 || max_ctx >> 31)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "tree_accept_in_cache: max_ctx = %zu out of range", max_ctx);
  return accept(tokens, parents, picked, n_seqs, n_tree, path, n_accepted, next_token, ctx_len, ctx_len_out, history,
                history_stride, max_ctx, stream);
}

WH_API int wh_kv_cache_compact(void* const* k_caches, void* const* v_caches, size_t n_layers, size_t n_seqs,
                               size_t max_ctx, size_t n_kv_heads, size_t head_dim, const uint32_t* path, size_t n_tree,
                               const uint32_t* n_accepted, const uint32_t* ctx_len, wh_stream_t stream) {
  // a row is at most 65535 workgroups of 256 pieces
  size_t row_bytes;
  if (__builtin_mul_overflow(n_kv_heads, head_dim, &row_bytes) || __builtin_mul_overflow(row_bytes, 2, &row_bytes) ||
      row_bytes == 0 || row_bytes % 16 != 0 || row_bytes >> 28)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "kv_cache_compact: rows of %zu x %zu f16 must be whole 16-byte pieces, below 2^28 bytes",
                         n_kv_heads, head_dim);
  if (n_tree > wh::kMaxTreeNodes || n_seqs > 65535 || max_ctx == 0 || max_ctx >> 31)
    return wh::set_error(WH_ERR_INVALID_SHAPE,
                         "kv_cache_compact: %zu nodes (at most %zu) of %zu sequences (at most 65535), max_ctx %zu", n_tree,
                         wh::kMaxTreeNodes, n_seqs, max_ctx);
  if (n_layers == 0 || n_seqs == 0 || n_tree == 0) return WH_OK;
  if (!k_caches || !v_caches || !path || !n_accepted || !ctx_len)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "kv_cache_compact: null pointer");
  if (!wh::aligned(path, 4) || !wh::aligned(n_accepted, 4) || !wh::aligned(ctx_len, 4))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "kv_cache_compact: arrays must be 4-byte aligned");
  for (size_t l = 0; l < n_layers; l++)
    if (!k_caches[l] || !v_caches[l] || !wh::aligned(k_caches[l], 16) || !wh::aligned(v_caches[l], 16))
      return wh::set_error(WH_ERR_INVALID_ARGUMENT,
                           "kv_cache_compact: layer %zu caches must be non-null and 16-byte aligned", l);
  // rows of a cache named twice, or shared by two, would be moved twice at once: in order of
  // their addresses every cache ends before the next begins
  size_t cache_bytes;
  if (__builtin_mul_overflow(n_seqs * max_ctx, row_bytes, &cache_bytes))
    return wh::set_error(WH_ERR_INVALID_SHAPE, "kv_cache_compact: %zu x %zu rows of %zu bytes are no cache", n_seqs, max_ctx,
                         row_bytes);
  uintptr_t few[4 * kCompactLayers];
  std::unique_ptr<uintptr_t[]> many;
  const size_t n_caches = 2 * n_layers;
  if (n_caches > 4 * kCompactLayers) many.reset(new (std::nothrow) uintptr_t[n_caches]);
  uintptr_t* at = many ? many.get() : few;
  if (n_caches > 4 * kCompactLayers && !many)
    return wh::set_error(WH_ERR_OOM, "kv_cache_compact: no memory for %zu caches", n_caches);
  for (size_t l = 0; l < n_layers; l++) {
    at[2 * l] = reinterpret_cast<uintptr_t>(k_caches[l]);
    at[2 * l + 1] = reinterpret_cast<uintptr_t>(v_caches[l]);
  }
  std::sort(at, at + n_caches);
  for (const size_t least : {static_cast<size_t>(1), cache_bytes})
    for (size_t i = 0; i + 1 < n_caches; i++)
      if (at[i + 1] - at[i] < least) {
        size_t l = n_layers - 1;
        while (reinterpret_cast<uintptr_t>(k_caches[l]) != at[i + 1] && reinterpret_cast<uintptr_t>(v_caches[l]) != at[i + 1]) l--;
        return least == 1
                   ? wh::set_error(WH_ERR_INVALID_ARGUMENT, "kv_cache_compact: a cache of layer %zu is named twice", l)
                   : wh::set_error(WH_ERR_INVALID_ARGUMENT,
                                   "kv_cache_compact: a cache of layer %zu begins within another (of %zu bytes)", l, cache_bytes);
      }
  CompactParams P{};
  P.path = path;
  P.n_accepted = n_accepted;
  P.ctx_len = ctx_len;
  P.max_ctx = max_ctx;
  P.row16 = static_cast<uint32_t>(row_bytes / 16);
  P.n_tree = static_cast<uint32_t>(n_tree);
  for (size_t l0 = 0; l0 < n_layers; l0 += kCompactLayers) {
    const size_t n = n_layers - l0 < kCompactLayers ? n_layers - l0 : kCompactLayers;
    for (size_t l = 0; l < n; l++) {
      P.cache[2 * l] = static_cast<piece16*>(k_caches[l0 + l]);
      P.cache[2 * l + 1] = static_cast<piece16*>(v_caches[l0 + l]);
    }
    const dim3 grid(static_cast<unsigned>(2 * n), static_cast<unsigned>(n_seqs), (P.row16 + 255) / 256);
    kv_compact_kernel<<<grid, 256, 0, reinterpret_cast<hipStream_t>(stream)>>>(P);
    WH_LAUNCH_CHECK("KV cache compaction launch");
  }
  return WH_OK;
}
