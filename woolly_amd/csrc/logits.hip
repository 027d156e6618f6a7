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
// One pass over the logits: a workgroup takes kChunk tokens of some rows of one
// sequence, counts the history's tokens that fall into them in LDS once, and per
// row adds the path's tokens, applies everything and reduces the highest token;
// a second small launch joins the chunks of a row.  Counting and the choice of a
// bias entry use integer LDS atomics (add, max): their order does not change the
// result.  Many rows are bound by memory: 64 nodes x 128256 (66.7 MB) take 19.3 us,
// 3.9 TB/s once the launch is under way.  With 2 rows per workgroup a call takes
// 20.3 us, with one 22.6, with four 23.4.  The rows go out past the L2, which would
// have them to write back when the kernel ends (21.0 us; 16 x 128256 10.6 against
// 9.5); loads past it gain nothing (20.4).  Workgroups of 2048, 4096 and 8192
// tokens, before that: 20.0, 19.3 and 19.6 us, but long histories, which every
// workgroup reads, favour large ones: 16 x 128256 with up to 20000 tokens each
// 14.2, 11.2 and 10.0.  One row of 32000 is the launch's latency: 5.8 us.
#include "tree.hpp"

namespace {

constexpr int kThreads = 1024;
constexpr int kChunk = 8192;  // tokens of a row per workgroup
constexpr int kPer = kChunk / kThreads;
constexpr uint32_t kNoToken = 0xFFFFFFFFu;
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Params {
  const float* logits;
  float* out;
  size_t ld, ldo;
  uint32_t vocab, rows_per_seq, rows_per_wg, n_chunks;
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
  float2* best;         // [n_rows][n_chunks] (logit, token's bits), null: no token wanted
  uint32_t* token;
};

// The highest token of some, as (logit, token): logit -inf and no token where
// there is none.
struct Best {
  float top;
  uint32_t at;
};
__device__ __forceinline__ Best wave_best(Best b) {
  const float m = whd::wave_max(b.top);
  return Best{m, whd::wave_min(b.top == m && m > -INFINITY ? b.at : kNoToken)};
}

// grid: (n_chunks, sequences * groups of rows_per_wg rows).  Thread t holds
// tokens 4 t .. 4 t + 3 and those 4096 behind them (VEC: rows 16-byte aligned), or
// tokens t, t + 1024, ...; `at` is the place of its j-th token in the chunk.
template <bool VEC>
__global__ __launch_bounds__(kThreads, 8) void logits_kernel(const Params P) {
#pragma clang fp contract(off)
  extern __shared__ __align__(16) uint32_t lds[];
  uint32_t* count = lds;                                   // [kChunk]
  int* entry = reinterpret_cast<int*>(lds + kChunk);       // [kChunk], with biases only
  __shared__ Best red[kThreads / 64];
  const uint32_t groups = (P.rows_per_seq + P.rows_per_wg - 1) / P.rows_per_wg;
  const uint32_t seq = blockIdx.y / groups, node0 = blockIdx.y % groups * P.rows_per_wg;
  const uint32_t nodes = min(P.rows_per_wg, P.rows_per_seq - node0);
  const uint32_t i0 = blockIdx.x * kChunk, n = min(P.vocab - i0, static_cast<uint32_t>(kChunk));
  const uint32_t t = threadIdx.x;
  auto at = [&](int j) -> uint32_t { return VEC ? 4 * t + (j & 3) + 4096 * (j >> 2) : t + kThreads * j; };
  float next[kPer];
  uint32_t next_open[kPer / 4];  // bit k: token at(4 q + k) exists and is allowed
  auto load = [&](size_t row) {
    const uint32_t* m = P.mask ? P.mask + row * P.mask_stride + i0 / 32 : nullptr;
#pragma unroll
    for (int q = 0; q < kPer / 4; q++) {
      if constexpr (VEC) {
        const uint32_t a = at(4 * q), left = a < n ? n - a : 0u;
        next_open[q] = (m && left ? m[a >> 5] >> (a & 31) : 15u) & (left < 4 ? (1u << left) - 1u : 15u);
      } else {
        next_open[q] = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t a = at(4 * q + k);
          if (a < n) next_open[q] |= (m ? m[a >> 5] >> (a & 31) & 1u : 1u) << k;
        }
      }
    }
    const float* p = P.logits + row * P.ld + i0;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < kPer; j += 4) {
        const uint32_t a = at(j);
        if (a + 4 <= n) {
          const float4 v = *reinterpret_cast<const float4*>(p + a);
          next[j] = v.x, next[j + 1] = v.y, next[j + 2] = v.z, next[j + 3] = v.w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; k++) next[j + k] = a + k < n ? p[a + k] : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; j++) next[j] = at(j) < n ? p[at(j)] : 0.f;
    }
  };
  const size_t row0 = static_cast<size_t>(seq) * P.rows_per_seq + node0;
  load(row0);
  whd::TreeLanes tree{};
  uint32_t node_token = 0;
  if (P.tree_parents) {
    tree = whd::tree_lanes(P.tree_parents + static_cast<size_t>(seq) * P.rows_per_seq, P.rows_per_seq);
    if (t < P.rows_per_seq) node_token = P.tree_tokens[static_cast<size_t>(seq) * P.rows_per_seq + t];
  }
  const bool said = P.history || P.tree_tokens;
#pragma unroll
  for (int j = 0; j < kChunk / 4 / kThreads; j++) {
    reinterpret_cast<uint4*>(count)[t + kThreads * j] = make_uint4(0, 0, 0, 0);
    if (P.n_bias) reinterpret_cast<int4*>(entry)[t + kThreads * j] = make_int4(-1, -1, -1, -1);
  }
  whd::lds_barrier();
  auto add = [&](uint32_t id) {
    if (id - i0 < n) atomicAdd(&count[id - i0], 1u);
  };
  if (P.history) {
    const uint32_t* h = P.history + seq * P.history_stride;
    // 16-byte loads from the first aligned entry on; the first ones do not wait for the length
    const size_t cap = P.history_stride, head = min(cap, (16 - (reinterpret_cast<uintptr_t>(h) & 15)) / 4 & 3);
    const size_t body = (cap - head) / 4, tail = head + 4 * body;
    const uint4* h4 = reinterpret_cast<const uint4*>(h + head);
    uint4 a = make_uint4(kNoToken, kNoToken, kNoToken, kNoToken), b = a;
    uint32_t c = kNoToken, d = kNoToken;
    if (t < body) a = h4[t];
    if (t + kThreads < body) b = h4[t + kThreads];
    if (t < head) c = h[t];
    if (tail + t < cap) d = h[tail + t];
    size_t len = cap;
    if (P.history_len && P.history_len[seq] < len) len = P.history_len[seq];
    auto add4 = [&](const uint4& v, size_t i) {
      if (i < len) add(v.x);
      if (i + 1 < len) add(v.y);
      if (i + 2 < len) add(v.z);
      if (i + 3 < len) add(v.w);
    };
    if (t < len) add(c);
    if (tail + t < len) add(d);
    for (size_t i = t;; i += 2 * kThreads) {
      const size_t next = i + 2 * kThreads;
      const uint4 u = a, v = b;
      if (head + 4 * next < len && next < body) a = h4[next];
      if (head + 4 * (next + kThreads) < len && next + kThreads < body) b = h4[next + kThreads];
      if (i < body) add4(u, head + 4 * i);
      if (i + kThreads < body) add4(v, head + 4 * (i + kThreads));
      if (next >= body || head + 4 * next >= len) break;
    }
  }
  for (uint32_t i = t; i < P.n_bias; i += kThreads) {
    const uint32_t c = P.bias_ids[seq * P.bias_stride + i] - i0;
    if (c < n) atomicMax(&entry[c], static_cast<int>(i));
  }
  const float* bias = P.bias + seq * P.bias_stride;
  for (uint32_t r = 0; r < nodes; r++) {
    const size_t row = row0 + r;
    bool present = true, mine = false;
    if (P.tree_parents) {
      const whd::TreePath path = whd::tree_path(tree, node0 + r);
      present = path.present();
      mine = t < P.rows_per_seq && path.has(t) && node_token - i0 < n;
      if (mine) atomicAdd(&count[node_token - i0], 1u);
    }
    whd::lds_barrier();  // the counts of this row
    Best best{-INFINITY, kNoToken};
    float x[kPer];
    uint32_t open[kPer / 4];
#pragma unroll
    for (int j = 0; j < kPer; j++) x[j] = next[j];
#pragma unroll
    for (int q = 0; q < kPer / 4; q++) open[q] = next_open[q];
    if (r + 1 < nodes) load(row + 1);
    if (present) {
      float* o = P.out ? P.out + row * P.ldo + i0 : nullptr;
#pragma unroll
      for (int q = 0; q < kPer / 4; q++) {
        float* l = x + 4 * q;
        if (said) {
          uint32_t c[4];
#pragma unroll
          for (int k = 0; k < 4; k++) c[k] = count[at(4 * q + k)];
          if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const float p = l[k] > 0.f ? l[k] / P.repetition : l[k] * P.repetition;
              const float f = static_cast<float>(c[k]) * P.frequency;
              l[k] = c[k] ? p - (f + P.presence) : l[k];
            }
          }
        }
        if (P.n_bias) {
          int e[4];
#pragma unroll
          for (int k = 0; k < 4; k++) e[k] = entry[at(4 * q + k)];
          if ((e[0] & e[1] & e[2] & e[3]) >= 0) {  // an entry's index is no negative number
#pragma unroll
            for (int k = 0; k < 4; k++)
              if (e[k] >= 0) l[k] = l[k] + bias[e[k]];
          }
        }
        if (open[q] != 15u) {
#pragma unroll
          for (int k = 0; k < 4; k++) l[k] = open[q] >> k & 1u ? l[k] : -INFINITY;
        }
        const float m = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));  // passes NaN over
        if (m > best.top) {  // at() grows with q and k: the lowest of equal ones
          best.top = m;
          best.at = i0 + at(4 * q + (l[0] == m ? 0 : l[1] == m ? 1 : l[2] == m ? 2 : 3));
        }
      }
      if (o) {
        if constexpr (VEC) {
#pragma unroll
          for (int j = 0; j < kPer; j += 4) {
            const uint32_t a = at(j);
            if (a + 4 <= n) {
              __builtin_nontemporal_store(f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]}, reinterpret_cast<f32x4*>(o + a));
            } else {
#pragma unroll
              for (int k = 0; k < 4; k++)
                if (a + k < n) o[a + k] = x[j + k];
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < kPer; j++)
            if (at(j) < n) o[at(j)] = x[j];
        }
      }
    }
    if (P.best) {
      best = wave_best(best);
      if ((t & 63) == 0) red[t >> 6] = best;
    }
    if (P.best || P.tree_parents) whd::lds_barrier();  // red, and every thread is done with the counts
    if (mine) atomicSub(&count[node_token - i0], 1u);
    if (P.best && t < 64) {
      best = wave_best(t < kThreads / 64 ? red[t] : Best{-INFINITY, kNoToken});
      if (t == 0) {
        if (P.n_chunks == 1) P.token[row] = best.at;
        else P.best[row * P.n_chunks + blockIdx.x] = make_float2(best.top, __builtin_bit_cast(float, best.at));
      }
    }
    whd::lds_barrier();  // red is free; the counts are the history's again
  }
}

// One wave per row.
__global__ __launch_bounds__(64) void logits_pick_kernel(const float2* __restrict__ best, uint32_t n_chunks,
                                                         uint32_t* __restrict__ token) {
  Best b{-INFINITY, kNoToken};
  for (uint32_t c = threadIdx.x; c < n_chunks; c += 64) {
    const float2 v = best[static_cast<size_t>(blockIdx.x) * n_chunks + c];
    if (v.x > b.top) b = Best{v.x, __builtin_bit_cast(uint32_t, v.y)};  // chunks ascend: so do their tokens
  }
  b = wave_best(b);
  if (threadIdx.x == 0) token[blockIdx.x] = b.at;
}

size_t chunks_of(size_t vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace

WH_API size_t wh_logits_process_workspace_bytes(const wh_logits_rules* rules, size_t n_rows, size_t vocab) {
  if (!rules) return 0;
  return n_rows * chunks_of(vocab) * sizeof(float2);
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
  if (r.n_bias && r.bias_stride && r.bias_stride < r.n_bias)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "logits_process: bias stride %zu below the %zu entries of a sequence",
                         r.bias_stride, r.n_bias);
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
  P.best = token ? static_cast<float2*>(workspace) : nullptr;
  P.token = token;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // rows of one sequence share the counts of a workgroup: as many as leave two workgroups per CU
  const size_t wgs = P.n_chunks * n_rows, most = 2 * static_cast<size_t>(wh::cu_count());
  P.rows_per_wg = static_cast<uint32_t>(wgs / most < 1 ? 1 : wgs / most < per ? wgs / most : per);
  const size_t groups = (per + P.rows_per_wg - 1) / P.rows_per_wg;
  const dim3 grid(P.n_chunks, static_cast<unsigned>(n_rows / per * groups));
  const size_t lds = kChunk * 4 * (P.n_bias ? 2 : 1);
  const bool vec = wh::aligned(logits, 16) && ld % 4 == 0 && (!out || (wh::aligned(out, 16) && ld_out % 4 == 0));
  if (vec) {
    WH_ENSURE_LDS(lds, &logits_kernel<true>);
    logits_kernel<true><<<grid, kThreads, lds, s>>>(P);
  } else {
    WH_ENSURE_LDS(lds, &logits_kernel<false>);
    logits_kernel<false><<<grid, kThreads, lds, s>>>(P);
  }
  WH_LAUNCH_CHECK("logits kernel launch");
  if (token && P.n_chunks > 1) {
    logits_pick_kernel<<<static_cast<unsigned>(n_rows), 64, 0, s>>>(P.best, P.n_chunks, token);
    WH_LAUNCH_CHECK("logits pick launch");
  }
  return WH_OK;
}
