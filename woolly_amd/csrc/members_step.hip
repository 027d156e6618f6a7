// members_step.hip -- one step of a Llama-shaped model for several continuations
// of the prompt in its caches: the decode step's layer (decode.hip) for all of
// them, with the rotation of rope.hip and the attention of shared_attention.hip.
#include "llama_step.hpp"
#include "members.hpp"

namespace {

constexpr const char* kFn = "llama_forward_members";

size_t attention_bytes(const wh_llama_model* m, size_t n_members, size_t max_own) {
  return wh::shared_attention_workspace_bytes(1, n_members, m->n_heads, m->n_kv_heads, m->head_dim, m->max_ctx, max_own);
}

}  // namespace

WH_API size_t wh_llama_forward_members_workspace_bytes(const wh_llama_model* model, size_t n_members, size_t max_own) {
  if (n_members == 0 || n_members > wh::kMaxTreeNodes || max_own == 0 || max_own >> 31 || check_model(kFn, model, false)) return 0;
  return step_layout(model, n_members, attention_bytes(model, n_members, max_own), nullptr).bytes;
}

WH_API int wh_llama_forward_members(const wh_llama_model* model, const wh_rope_rules* rules, const uint32_t* tokens,
                                    size_t n_members, const uint32_t* prefix_len, const uint32_t* len,
                                    void* const* k_own, void* const* v_own, size_t max_own, float* x, float* logits,
                                    void* workspace, size_t workspace_bytes, wh_stream_t stream) {
  int st = check_model(kFn, model, logits != nullptr);
  if (st) return st;
  if (n_members > wh::kMaxTreeNodes)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: %zu members (at most %zu)", kFn, n_members, wh::kMaxTreeNodes);
  if (max_own == 0 || max_own >> 31)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: max_own = %zu out of range", kFn, max_own);
  wh_rope_rules rope{};
  rope.inv_freq = model->rope_inv_freq;
  if (rules) rope = *rules;
  if ((st = wh::check_rope_rules(kFn, rope, model->head_dim))) return st;
  if (n_members == 0) return WH_OK;
  if (!tokens || !prefix_len || !len || !x || !k_own || !v_own)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null pointer", kFn);
  if (!wh::aligned(prefix_len, 4) || !wh::aligned(len, 4) || !wh::aligned(logits, 4))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: arrays must be 4-byte aligned", kFn);
  for (size_t l = 0; l < model->n_layers; l++)
    if (!k_own[l] || !v_own[l] || k_own[l] == v_own[l] || !wh::aligned(k_own[l], 16) || !wh::aligned(v_own[l], 16))
      return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: layer %zu own caches must be non-null, two and 16-byte aligned", kFn, l);
  if (!model->token_embd) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: the model has no token_embd table", kFn);
  if ((st = wh::check_embedding_args(kFn, model->token_embd_type, model->token_embd, model->vocab, model->hidden, tokens, x)))
    return st;
  const Ws w = step_layout(model, n_members, attention_bytes(model, n_members, max_own), workspace);
  if (!workspace || workspace_bytes < w.bytes)
    return wh::set_error(WH_ERR_BUFFER_TOO_SMALL, "%s: workspace too small: needed %zu bytes, available %zu", kFn, w.bytes,
                         workspace ? workspace_bytes : static_cast<size_t>(0));
  if (!wh::aligned(workspace, 256))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: workspace is not 256-byte aligned", kFn);
  const size_t heads = model->n_heads, kv = model->n_kv_heads, D = model->head_dim, qd = heads * D, kvd = kv * D;
  return run_step(model, tokens, n_members, x, logits, w, stream, [&](size_t l, const Ws& w, hipStream_t s) {
    const wh_llama_layer& L = model->layers[l];
    const wh::RopeArgs r{w.q, w.k, w.v, qd, kvd, prefix_len, len, n_members, n_members, 1, heads,
                         kv, D, w.q, qd, nullptr, 0, k_own[l], v_own[l], max_own};
    const int st = wh::launch_rope(rope, r, s);
    if (st) return st;
    const wh::SharedAttnArgs a{w.q, qd, prefix_len, len, 1, n_members, L.k_cache, L.v_cache, model->max_ctx,
                               k_own[l], v_own[l], max_own, heads, kv, D, w.attn};
    return wh::launch_shared_attention(a, w.att_ws, s);
  });
}
