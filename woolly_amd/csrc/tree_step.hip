// tree_step.hip -- one step of a Llama-shaped model for every node of a tree of
// drafted tokens: the decode step's layer (decode.hip) for n_tree tokens, with
// the attention of tree_attention.hip.
#include "llama_step.hpp"

namespace {

size_t attention_bytes(const wh_llama_model* m, size_t n_tree) {
  return wh::tree_attention_workspace_bytes(1, n_tree, m->n_heads, m->n_kv_heads, m->head_dim, m->max_ctx);
}

}  // namespace

WH_API size_t wh_llama_forward_tree_workspace_bytes(const wh_llama_model* model, size_t n_tree) {
  if (n_tree == 0 || n_tree > wh::kMaxTreeNodes || check_model("llama_forward_tree", model, false)) return 0;
  return step_layout(model, n_tree, attention_bytes(model, n_tree), nullptr).bytes;
}

WH_API int wh_llama_forward_tree(const wh_llama_model* model, const uint32_t* tokens, const int32_t* parents,
                                 size_t n_tree, const uint32_t* ctx_len, float* x, float* logits, void* workspace,
                                 size_t workspace_bytes, wh_stream_t stream) {
  int st = check_model("llama_forward_tree", model, logits != nullptr);
  if (st) return st;
  if (n_tree > wh::kMaxTreeNodes)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "llama_forward_tree: %zu nodes (at most %zu)", n_tree, wh::kMaxTreeNodes);
  if (n_tree == 0) return WH_OK;
  if (!tokens || !parents || !ctx_len || !x)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: null pointer");
  if (!wh::aligned(parents, 4) || !wh::aligned(ctx_len, 4) || !wh::aligned(logits, 4))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: arrays must be 4-byte aligned");
  if (!model->token_embd)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: the model has no token_embd table");
  if ((st = wh::check_embedding_args("llama_forward_tree", model->token_embd_type, model->token_embd, model->vocab,
                                     model->hidden, tokens, x)))
    return st;
  const Ws w = step_layout(model, n_tree, attention_bytes(model, n_tree), workspace);
  if (!workspace || workspace_bytes < w.bytes)
    return wh::set_error(WH_ERR_BUFFER_TOO_SMALL,
                         "llama_forward_tree: workspace too small: needed %zu bytes, available %zu", w.bytes,
                         workspace ? workspace_bytes : static_cast<size_t>(0));
  if (!wh::aligned(workspace, 256))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: workspace is not 256-byte aligned");
  const size_t D = model->head_dim, qd = model->n_heads * D, kvd = model->n_kv_heads * D;
  return run_step(model, tokens, n_tree, x, logits, w, stream, [&](size_t l, const Ws& w, hipStream_t s) {
    const wh_llama_layer& L = model->layers[l];
    const wh::TreeAttnArgs a{w.q, w.k, w.v, qd, kvd, parents, ctx_len, 1, n_tree, L.k_cache, L.v_cache,
                             model->max_ctx, model->n_heads, model->n_kv_heads, D, model->rope_inv_freq, w.attn};
    return wh::launch_tree_attention(a, w.att_ws, s);
  });
}
