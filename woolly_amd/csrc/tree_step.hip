// tree_step.hip -- one step of a Llama-shaped model for every node of a tree of
// drafted tokens: the decode step's layer (decode.hip) for n_tree tokens, with
// the attention of tree_attention.hip.
//
// One layer: x_hat = rms_norm(x); q, k, v = W x_hat (the several-token GEMMs); tree
// attention; x += Wo attn; x += FFN(x) (the fused layer of wh_ffn_swiglu where
// gate, up and down have one type, else the same in steps).  Nothing here
// allocates or synchronises, so a caller can capture the step into a HIP graph.
#include "tree.hpp"

namespace {

constexpr int kAddThreads = 256;

// x += y, n elements
__global__ __launch_bounds__(kAddThreads) void tree_add_kernel(float* __restrict__ x, const float* __restrict__ y, size_t n) {
  const size_t i = static_cast<size_t>(blockIdx.x) * kAddThreads + threadIdx.x;
  if (i < n) x[i] += y[i];
}

int launch_add(float* x, const float* y, size_t n, hipStream_t s) {
  tree_add_kernel<<<static_cast<unsigned>((n + kAddThreads - 1) / kAddThreads), kAddThreads, 0, s>>>(x, y, n);
  WH_LAUNCH_CHECK("residual add launch");
  return WH_OK;
}

size_t al256(size_t v) { return (v + 255) / 256 * 256; }
size_t max2(size_t a, size_t b) { return a > b ? a : b; }

// A layer's matrices in the order q k v o gate up down.
struct Mat {
  int type;
  const void* w;
  size_t rows, k;
};
struct LayerMats {
  Mat m[7];
};
LayerMats layer_mats(const wh_llama_model* m, const wh_llama_layer& L) {
  auto t = [&](int v) { return v ? v : m->type; };
  const size_t qd = m->n_heads * m->head_dim, kvd = m->n_kv_heads * m->head_dim;
  return {{{t(L.wq_type), L.wq, qd, m->hidden},
           {t(L.wk_type), L.wk, kvd, m->hidden},
           {t(L.wv_type), L.wv, kvd, m->hidden},
           {t(L.wo_type), L.wo, m->hidden, qd},
           {t(L.w_gate_type), L.w_gate, m->n_ff, m->hidden},
           {t(L.w_up_type), L.w_up, m->n_ff, m->hidden},
           {t(L.w_down_type), L.w_down, m->hidden, m->n_ff}}};
}
bool fused_ffn(const LayerMats& l) { return l.m[4].type == l.m[5].type && l.m[4].type == l.m[6].type; }

struct Ws {
  float *xn, *q, *k, *v, *attn, *y, *g, *u;
  void *att_ws, *gemm_ws;
  size_t gemm_bytes, bytes;
};

Ws layout(const wh_llama_model* m, size_t T, void* base) {
  Ws w{};
  char* b = static_cast<char*>(base);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    void* r = b ? b + off : nullptr;
    off += al256(bytes);
    return r;
  };
  const size_t qd = m->n_heads * m->head_dim, kvd = m->n_kv_heads * m->head_dim;
  auto floats = [&](size_t n) { return static_cast<float*>(take(4 * T * n)); };
  w.xn = floats(m->hidden);
  w.q = floats(qd);
  w.k = floats(kvd);
  w.v = floats(kvd);
  w.attn = floats(qd);
  w.y = floats(m->hidden);
  w.att_ws = take(wh::tree_attention_workspace_bytes(1, T, m->n_heads, m->n_kv_heads, m->head_dim, m->max_ctx));
  // one region for whichever product or feed-forward layer needs most
  size_t need = m->output ? wh::gemm_workspace_bytes_for(m->output_type, m->vocab, T, m->hidden) : 0;
  bool steps = false;
  for (size_t i = 0; i < m->n_layers; i++) {
    const LayerMats l = layer_mats(m, m->layers[i]);
    for (const Mat& a : l.m) need = max2(need, wh::gemm_workspace_bytes_for(a.type, a.rows, T, a.k));
    if (fused_ffn(l)) need = max2(need, wh_ffn_workspace_bytes_for_type(l.m[4].type, m->hidden, m->n_ff, T));
    else steps = true;
  }
  if (steps) {
    w.g = floats(m->n_ff);
    w.u = floats(m->n_ff);
  }
  w.gemm_bytes = al256(need);
  w.gemm_ws = take(need);
  w.bytes = off;
  return w;
}

int check_matrix(const char* what, const Mat& a) {
  if (!wh::is_block_type(a.type) && !wh::is_kquant(a.type))
    return wh::set_error(WH_ERR_UNSUPPORTED_TYPE, "llama_forward_tree: %s has unsupported ggml type %d", what, a.type);
  const size_t be = wh::block_elems(a.type);
  if (a.k % be != 0)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "llama_forward_tree: %s rows of %zu are not whole blocks of %zu", what, a.k, be);
  if (!a.w) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: %s is a null pointer", what);
  return WH_OK;
}

int check_model(const wh_llama_model* m, bool head) {
  if (!m || !m->layers || !m->rope_inv_freq)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: null model, layers or rope_inv_freq");
  if (m->hidden == 0 || m->n_ff == 0 || m->max_ctx == 0 || m->max_ctx >> 31)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "llama_forward_tree: hidden %zu, n_ff %zu, max_ctx %zu out of range", m->hidden,
                         m->n_ff, m->max_ctx);
  if (!wh::tree_attention_shape_ok(m->n_heads, m->n_kv_heads, m->head_dim))
    return wh::set_error(WH_ERR_INVALID_SHAPE, "llama_forward_tree: head_dim %zu, %zu heads, %zu KV heads not supported",
                         m->head_dim, m->n_heads, m->n_kv_heads);
  static const char* const names[7] = {"wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down"};
  for (size_t l = 0; l < m->n_layers; l++) {
    const wh_llama_layer& L = m->layers[l];
    const LayerMats mats = layer_mats(m, L);
    for (int i = 0; i < 7; i++) {
      const int st = check_matrix(names[i], mats.m[i]);
      if (st) return st;
    }
    if (!L.attn_norm || !L.ffn_norm || !L.k_cache || !L.v_cache || !wh::aligned(L.attn_norm, 4) ||
        !wh::aligned(L.ffn_norm, 4) || !wh::aligned(L.k_cache, 16) || !wh::aligned(L.v_cache, 16))
      return wh::set_error(WH_ERR_INVALID_ARGUMENT,
                           "llama_forward_tree: layer %zu norms (4-byte) and KV caches (16-byte aligned) must be non-null", l);
  }
  if (!head) return WH_OK;
  if (m->vocab == 0 || m->vocab >> 30)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "llama_forward_tree: vocab = %zu out of range", m->vocab);
  if (!m->output_norm) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: null output_norm");
  return check_matrix("output", {m->output_type, m->output, m->vocab, m->hidden});
}

}  // namespace

WH_API size_t wh_llama_forward_tree_workspace_bytes(const wh_llama_model* model, size_t n_tree) {
  if (n_tree == 0 || n_tree > wh::kMaxTreeNodes || check_model(model, false)) return 0;
  return layout(model, n_tree, nullptr).bytes;
}

WH_API int wh_llama_forward_tree(const wh_llama_model* model, const uint32_t* tokens, const int32_t* parents,
                                 size_t n_tree, const uint32_t* ctx_len, float* x, float* logits, void* workspace,
                                 size_t workspace_bytes, wh_stream_t stream) {
  int st = check_model(model, logits != nullptr);
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
  const Ws w = layout(model, n_tree, workspace);
  if (!workspace || workspace_bytes < w.bytes)
    return wh::set_error(WH_ERR_BUFFER_TOO_SMALL,
                         "llama_forward_tree: workspace too small: needed %zu bytes, available %zu", w.bytes,
                         workspace ? workspace_bytes : static_cast<size_t>(0));
  if (!wh::aligned(workspace, 256))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "llama_forward_tree: workspace is not 256-byte aligned");
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const size_t T = n_tree, H = model->hidden, F = model->n_ff, D = model->head_dim;
  const size_t qd = model->n_heads * D, kvd = model->n_kv_heads * D;
  auto gemm = [&](const Mat& a, const float* in, float* out) {
    return wh::launch_gemm(a.type, a.w, a.rows, a.k, in, T, out, w.gemm_ws, w.gemm_bytes, s);
  };
  if ((st = wh::launch_embedding_lookup(model->token_embd_type, model->token_embd, model->vocab, H, tokens, T, x, s)))
    return st;
  for (size_t l = 0; l < model->n_layers; l++) {
    const wh_llama_layer& L = model->layers[l];
    const LayerMats mats = layer_mats(model, L);
    if ((st = wh::launch_rms_norm(x, L.attn_norm, model->eps, T, H, w.xn, s))) return st;
    if ((st = gemm(mats.m[0], w.xn, w.q)) || (st = gemm(mats.m[1], w.xn, w.k)) || (st = gemm(mats.m[2], w.xn, w.v)))
      return st;
    const wh::TreeAttnArgs a{w.q, w.k, w.v, qd, kvd, parents, ctx_len, 1, T, L.k_cache, L.v_cache,
                             model->max_ctx, model->n_heads, model->n_kv_heads, D, model->rope_inv_freq, w.attn};
    if ((st = wh::launch_tree_attention(a, w.att_ws, s))) return st;
    if ((st = gemm(mats.m[3], w.attn, w.y)) || (st = launch_add(x, w.y, T * H, s))) return st;
    if (fused_ffn(mats)) {
      const wh_ffn_weights f{mats.m[4].type, mats.m[4].w, mats.m[5].w, mats.m[6].w, H, F};
      if ((st = wh_ffn_swiglu(&f, L.ffn_norm, model->eps, x, T, w.y, w.gemm_ws, w.gemm_bytes, stream))) return st;
    } else {
      if ((st = wh::launch_rms_norm(x, L.ffn_norm, model->eps, T, H, w.xn, s))) return st;
      if ((st = gemm(mats.m[4], w.xn, w.g)) || (st = gemm(mats.m[5], w.xn, w.u))) return st;
      if ((st = wh::launch_swiglu(w.g, w.u, T * F, w.g, s)) || (st = gemm(mats.m[6], w.g, w.y))) return st;
    }
    if ((st = launch_add(x, w.y, T * H, s))) return st;
  }
  if (!logits) return WH_OK;
  if ((st = wh::launch_rms_norm(x, model->output_norm, model->eps, T, H, w.xn, s))) return st;
  return gemm({model->output_type, model->output, model->vocab, H}, w.xn, logits);
}
