// logits.hip -- penalties for repeated tokens, biases and grammar masks on
// logits, and the highest token of each row, on gfx950.
//
// For logit l of token i in a row, with c the number of times i occurs in the
// row's history (its sequence's tokens and, for a node of a tree of drafted
// tokens, the tokens on the path to it):
//   c > 0:  l = l > 0 ? l / repetition : l * repetition
//           l = l - (c * frequency + presence)
//   l = l + bias[i]        (of several entries for i the last one counts)
//   l = -inf               where the row's mask has bit i clear
//   token = the lowest i with the largest l > -inf that is no NaN; none: all bits set
// Every operation is rounded by itself, in this order (no fused multiply-add),
// so the values do not depend on how the row is cut up.
//
// One pass over the logits: a workgroup takes kChunk tokens of a row, counts
// the history's tokens that fall into them in LDS, applies everything and
// reduces its highest token; a second small launch joins the chunks of a row.
// Counting and the choice of a bias entry use integer LDS atomics (add, max):
// their order does not change the result.
#include "tree.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 2048;  // tokens of a row per workgroup
constexpr uint32_t kNoToken = 0xFFFFFFFFu;

struct Params {
  const float* logits;
  float* out;
  size_t ld, ldo;
  uint32_t vocab, rows_per_seq, n_chunks;
  const uint32_t* history;
  size_t history_stride;
  const uint32_t* history_len;
  const uint32_t* tree_tokens;
  const int32_t* tree_parents;
  float repetition, frequency, presence;
  const uint32_t* bias_ids;
  const float* bias;
  uint32_t n_bias;
  size_t bias_stride;
  const uint32_t* mask;
  size_t mask_stride;
  unsigned long long* best;  // [n_rows][n_chunks], null: no token wanted
  uint32_t* token;
};

// Orders floats as unsigned integers (-0 as +0); NaN and -inf give 0: no candidate.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const unsigned long long o = __shfl_xor(v, off, 64);
    v = o > v ? o : v;
  }
  return v;
}

// grid: (n_chunks, n_rows)
__global__ __launch_bounds__(kThreads) void logits_kernel(const Params P) {
#pragma clang fp contract(off)
  __shared__ uint32_t count[kChunk];
  __shared__ int entry[kChunk];
  __shared__ unsigned long long red[kThreads / 64];
  const uint32_t row = blockIdx.y, seq = row / P.rows_per_seq, node = row % P.rows_per_seq;
  const uint32_t i0 = blockIdx.x * kChunk, n = min(P.vocab - i0, static_cast<uint32_t>(kChunk));
  const uint32_t t = threadIdx.x;
  const bool said = P.history || P.tree_tokens;
  for (int i = t; i < kChunk; i += kThreads) {
    count[i] = 0;
    entry[i] = -1;
  }
  __syncthreads();
  bool present = true;
  if (P.tree_parents) {
    const whd::TreePath path =
        whd::tree_path(P.tree_parents + static_cast<size_t>(seq) * P.rows_per_seq, P.rows_per_seq, node);
    present = path.present();
    if (t < P.rows_per_seq && path.has(t)) {
      const uint32_t c = P.tree_tokens[static_cast<size_t>(seq) * P.rows_per_seq + t] - i0;
      if (c < n) atomicAdd(&count[c], 1u);
    }
  }
  if (!present) {
    if (t == 0 && P.best) P.best[static_cast<size_t>(row) * P.n_chunks + blockIdx.x] = 0;
    return;
  }
  if (P.history) {
    const uint32_t* h = P.history + seq * P.history_stride;
    size_t len = P.history_stride;
    if (P.history_len && P.history_len[seq] < len) len = P.history_len[seq];
    for (size_t i = t; i < len; i += kThreads) {
      const uint32_t c = h[i] - i0;
      if (c < n) atomicAdd(&count[c], 1u);
    }
  }
  for (uint32_t i = t; i < P.n_bias; i += kThreads) {
    const uint32_t c = P.bias_ids[seq * P.bias_stride + i] - i0;
    if (c < n) atomicMax(&entry[c], static_cast<int>(i));
  }
  __syncthreads();
  const float* x = P.logits + row * P.ld + i0;
  float* o = P.out ? P.out + row * P.ldo + i0 : nullptr;
  const uint32_t* mask = P.mask ? P.mask + row * P.mask_stride + i0 / 32 : nullptr;
  unsigned long long best = 0;
  for (uint32_t i = t; i < n; i += kThreads) {
    float l = x[i];
    if (said) {
      const uint32_t c = count[i];
      if (c) {
        l = l > 0.f ? l / P.repetition : l * P.repetition;
        const float f = static_cast<float>(c) * P.frequency;
        l = l - (f + P.presence);
      }
    }
    if (P.n_bias) {
      const int e = entry[i];
      if (e >= 0) l = l + P.bias[seq * P.bias_stride + e];
    }
    if (mask && !((mask[i >> 5] >> (i & 31)) & 1u)) l = -INFINITY;
    if (o) o[i] = l;
    const uint32_t key = order_key(l);
    const unsigned long long b = static_cast<unsigned long long>(key) << 32 | (kNoToken - (i0 + i));
    if (key && b > best) best = b;
  }
  if (!P.best) return;
  best = wave_max(best);
  if ((t & 63) == 0) red[t >> 6] = best;
  __syncthreads();
  if (t == 0) {
    for (int w = 1; w < kThreads / 64; w++) best = red[w] > best ? red[w] : best;
    P.best[static_cast<size_t>(row) * P.n_chunks + blockIdx.x] = best;
  }
}

// One wave per row.
__global__ __launch_bounds__(64) void logits_pick_kernel(const unsigned long long* __restrict__ best, uint32_t n_chunks,
                                                         uint32_t* __restrict__ token) {
  unsigned long long b = 0;
  for (uint32_t c = threadIdx.x; c < n_chunks; c += 64) {
    const unsigned long long v = best[static_cast<size_t>(blockIdx.x) * n_chunks + c];
    b = v > b ? v : b;
  }
  b = wave_max(b);
  if (threadIdx.x == 0) token[blockIdx.x] = b ? kNoToken - static_cast<uint32_t>(b) : kNoToken;
}

size_t chunks_of(size_t vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace

WH_API size_t wh_logits_process_workspace_bytes(const wh_logits_rules* rules, size_t n_rows, size_t vocab) {
  if (!rules) return 0;
  return n_rows * chunks_of(vocab) * sizeof(unsigned long long);
}

WH_API int wh_logits_process(const wh_logits_rules* rules, const float* logits, size_t ld, size_t n_rows, size_t vocab,
                             float* out, size_t ld_out, uint32_t* token, void* workspace, size_t workspace_bytes,
                             wh_stream_t stream) {
  if (!rules) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "logits_process: null rules");
  const wh_logits_rules& r = *rules;
  const size_t per = r.rows_per_seq ? r.rows_per_seq : 1;
  if (vocab == 0 || vocab >= (static_cast<size_t>(1) << 31) || n_rows > 65535 || n_rows % per != 0)
    return wh::set_error(WH_ERR_INVALID_SHAPE,
                         "logits_process: %zu rows (at most 65535) of %zu logits, %zu rows per sequence", n_rows, vocab, per);
  if (ld < vocab || (out && ld_out < vocab) || (r.mask && r.mask_stride < (vocab + 31) / 32))
    return wh::set_error(WH_ERR_INVALID_SHAPE,
                         "logits_process: strides %zu, %zu and %zu mask words below the rows' %zu logits", ld, ld_out,
                         r.mask_stride, vocab);
  if ((r.tree_tokens != nullptr) != (r.tree_parents != nullptr) || (r.tree_tokens && per > wh::kMaxTreeNodes))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT,
                         "logits_process: a tree has tokens and parents, and at most %zu nodes (here %zu)",
                         wh::kMaxTreeNodes, per);
  if (!(r.repetition_penalty > 0.f && r.repetition_penalty <= 3.402823466e38f) ||
      !(r.frequency_penalty - r.frequency_penalty == 0.f) || !(r.presence_penalty - r.presence_penalty == 0.f))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT,
                         "logits_process: the repetition penalty must be finite and above 0, the others finite");
  if (r.n_bias && (!r.bias_ids || !r.bias || r.n_bias >> 31))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "logits_process: %zu bias entries without ids or values", r.n_bias);
  if (n_rows == 0 || (!out && !token)) return WH_OK;
  if (!logits) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "logits_process: null logits");
  if (out == logits && ld_out != ld)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "logits_process: in place, both strides must be the same");
  const void* ptrs[] = {logits, out, token, r.history, r.history_len, r.tree_tokens, r.tree_parents, r.bias_ids, r.bias, r.mask};
  for (const void* p : ptrs)
    if (!wh::aligned(p, 4))
      return wh::set_error(WH_ERR_INVALID_ARGUMENT, "logits_process: arrays must be 4-byte aligned");
  const size_t need = token ? wh_logits_process_workspace_bytes(rules, n_rows, vocab) : 0;
  if (workspace_bytes < need || (need && !workspace))
    return wh::set_error(WH_ERR_BUFFER_TOO_SMALL, "logits_process: workspace too small: needed %zu bytes, available %zu",
                         need, workspace ? workspace_bytes : static_cast<size_t>(0));
  if (need && !wh::aligned(workspace, 8))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "logits_process: the workspace must be 8-byte aligned");
  Params P{};
  P.logits = logits, P.ld = ld;
  P.out = out, P.ldo = ld_out;
  P.vocab = static_cast<uint32_t>(vocab);
  P.rows_per_seq = static_cast<uint32_t>(per);
  P.n_chunks = static_cast<uint32_t>(chunks_of(vocab));
  // penalties that change nothing need no counts; an absent node's row is left alone all the same
  const bool penal = r.repetition_penalty != 1.f || r.frequency_penalty != 0.f || r.presence_penalty != 0.f;
  if (penal && r.history && r.history_stride) {
    P.history = r.history;
    P.history_stride = r.history_stride;
    P.history_len = r.history_len;
  }
  P.tree_tokens = r.tree_tokens;
  P.tree_parents = r.tree_parents;
  P.repetition = r.repetition_penalty;
  P.frequency = r.frequency_penalty;
  P.presence = r.presence_penalty;
  if (r.n_bias) {
    P.bias_ids = r.bias_ids;
    P.bias = r.bias;
    P.n_bias = static_cast<uint32_t>(r.n_bias);
    P.bias_stride = r.bias_stride;
  }
  P.mask = r.mask;
  P.mask_stride = r.mask_stride;
  P.best = token ? static_cast<unsigned long long*>(workspace) : nullptr;
  P.token = token;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  logits_kernel<<<dim3(P.n_chunks, static_cast<unsigned>(n_rows)), kThreads, 0, s>>>(P);
  WH_LAUNCH_CHECK("logits kernel launch");
  if (token) {
    logits_pick_kernel<<<static_cast<unsigned>(n_rows), 64, 0, s>>>(P.best, P.n_chunks, token);
    WH_LAUNCH_CHECK("logits pick launch");
  }
  return WH_OK;
}
