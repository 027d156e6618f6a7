// rope.hip -- norms of queries and keys per head, their rotation by position,
// and the new rows of the f16 KV caches, in one pass, on gfx950.
//
// Token i of a member (the n_new new ones are its last) has position
// p = base_len + i.  Per head of d elements, each step where it is wanted:
//   x = x / sqrt(sum x^2 / d + eps) * w
//   (x, y) = c (x cos a - y sin a, x sin a + y cos a),  a = p inv_freq[j]
// for the pairs (j, j + r / 2), or (2 j, 2 j + 1), j < r / 2, of its first r
// elements.  q goes out in f32, k and v to row i of the member's caches.
//
// The angle is formed in 64 bits, as turns, of which only the part behind the
// point is kept: in 32 bits p * inv_freq would be off by p 2^-24 radians.  Its
// sine and cosine are of that part, in 64 bits; k is normed and turned in 64 bits
// and rounded to f32, then to f16, so a cache row is what the formula gives (and
// what wh_attention_tree stores), q in 32 (its norm in 64 where the mean square is
// no normal f32 number).
//
// Many rows are bound by memory: 4000 of 32 / 8 heads of 128, 180 MB read and
// written, 35.5 us, normed 42 (5.1 and 4.3 TB/s); few by the launch and two loads
// one behind the other: 8 rows 3.1 us in a graph.
#include <type_traits>

#include "members.hpp"
#include "tree.hpp"

namespace {

constexpr int kThreads = 256;
constexpr size_t kGridWidth = 1 << 22;  // a launch has fewer than 2^32 threads in a dimension
constexpr size_t kManyHeads = 8192;  // heads of all rows from which on a wave takes more turns
struct Params {
  const float *q, *k, *v;
  size_t ldq, ldkv, ldq_out, ldk_out, max_rows;
  const uint32_t *base_len, *len;
  const float *inv_freq, *q_norm, *k_norm;
  float *q_out, *k_out;
  _Float16 *k_cache, *v_cache;
  uint32_t n_per, n_new, n_heads, n_kv, d, half, groups, rows;  // half: turned pairs
  int interleaved;
  float eps;
  double per_d, magnitude;  // 1 / d
};

// A 64-bit value as the cache holds it: rounded to f32, then to f16.  (The
// empty statement keeps the compiler from joining the two into one rounding.)
__device__ __forceinline__ _Float16 stored(double x) {
  float f = static_cast<float>(x);
  asm("" : "+v"(f));
  return static_cast<_Float16>(f);
}

// Sum over the L lanes (32 or 64) that share a head, in every one of them.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});
  v += dpp(v, std::integral_constant<int, 0x4E>{});
  v += dpp(v, std::integral_constant<int, 0x141>{});
  v += dpp(v, std::integral_constant<int, 0x140>{});
  const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  v = __builtin_bit_cast(float, static_cast<uint32_t>(a[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(a[1]));
  if constexpr (L == 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = __builtin_bit_cast(float, static_cast<uint32_t>(b[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(b[1]));
  }
  return v;
}

// A wave takes N turns of 64 / L heads of one row, the query heads first, then
// the key heads with their values.  A lane has PP pairs of its head: pair
// l + L u, turned ones first, then (in two halves) the rest of the head.
// grid: rows * groups of heads, in rows of kGridWidth workgroups.
template <int L, int PP, int N>
__global__ __launch_bounds__(kThreads) void rope_kernel(const Params P) {
  constexpr uint32_t kHeads = 64 / L * N;
  const uint32_t lane = threadIdx.x & 63, l = lane % L;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t item = (blockIdx.y * gridDim.x + blockIdx.x) * (kThreads / 64) + wave;
  const uint32_t row = item / P.groups, group = item % P.groups;  // row: member * n_new + token
  const uint32_t n_slots = P.n_heads + P.n_kv;
  const uint32_t h0 = group * kHeads + (L == 32 ? lane / 32 : 0);
  if (row >= P.rows) return;
  const uint32_t m = row / P.n_new, t = row % P.n_new;
  const bool any_k = group * kHeads + kHeads > P.n_heads;

  uint32_t a[PP], b[PP];  // the two elements of a pair
  bool in[PP], turned[PP];
#pragma unroll
  for (int u = 0; u < PP; u++) {
    const uint32_t i = l + L * u;
    in[u] = i < P.d / 2;
    turned[u] = i < P.half;
    const uint32_t rest = P.half + i;  // element 2 half + (i - half)
    a[u] = turned[u] ? (P.interleaved ? 2 * i : i) : rest;
    b[u] = turned[u] ? (P.interleaved ? 2 * i + 1 : i + P.half) : rest + P.d / 2 - P.half;
    if (!in[u]) a[u] = b[u] = 0;
  }
  float x[N][PP], y[N][PP], vx[N][PP], vy[N][PP];
#pragma unroll
  for (int n = 0; n < N; n++) {
    const uint32_t h = min(h0 + n * (64 / L), n_slots - 1);
    const bool is_q = h < P.n_heads;
    const size_t at = static_cast<size_t>(is_q ? h : h - P.n_heads) * P.d;
    const float* src = (is_q ? P.q + row * P.ldq : P.k + row * P.ldkv) + at;
#pragma unroll
    for (int u = 0; u < PP; u++) {
      x[n][u] = src[a[u]];
      y[n][u] = src[b[u]];
      vx[n][u] = vy[n][u] = 0.f;
      if (!is_q && P.v_cache) {
        const float* v = P.v + row * P.ldkv + at;
        vx[n][u] = v[a[u]];
        vy[n][u] = v[b[u]];
      }
    }
  }
  const uint32_t len = P.len ? P.len[m] : P.n_new;
  const uint32_t base = P.base_len ? P.base_len[m / P.n_per] : 0;
  const long long i = static_cast<long long>(len) - P.n_new + t;  // the member's token
  const bool present = i >= 0, fits = !P.k_cache || i < static_cast<long long>(P.max_rows);
  double cs[PP], sn[PP];
  float qw[PP][2], kw[PP][2];
#pragma unroll
  for (int u = 0; u < PP; u++) {
    cs[u] = sn[u] = 0.0;
    if (turned[u]) {
      const double inv = static_cast<double>(P.inv_freq[l + L * u]);
      const double turns = (static_cast<double>(base) + static_cast<double>(i)) * inv * 0.15915494309189535;
      sincospi(2.0 * (turns - rint(turns)), &sn[u], &cs[u]);
      cs[u] *= P.magnitude;
      sn[u] *= P.magnitude;
    }
    qw[u][0] = P.q_norm ? P.q_norm[a[u]] : 1.f;
    qw[u][1] = P.q_norm ? P.q_norm[b[u]] : 1.f;
    kw[u][0] = P.k_norm && any_k ? P.k_norm[a[u]] : 1.f;
    kw[u][1] = P.k_norm && any_k ? P.k_norm[b[u]] : 1.f;
  }
#pragma unroll
  for (int n = 0; n < N; n++) {
    const uint32_t h = h0 + n * (64 / L);
    const bool is_q = h < P.n_heads;
    double kx[PP], ky[PP];  // of a key head
    auto root64 = [&]() __attribute__((always_inline)) {  // 1 / sqrt(mean square + eps)
      double sum = 0.0;
#pragma unroll
      for (int u = 0; u < PP; u++) {
        const double dx = in[u] ? x[n][u] : 0.f, dy = in[u] ? y[n][u] : 0.f;
        sum = __builtin_fma(dx, dx, __builtin_fma(dy, dy, sum));
      }
      const double mean = __builtin_fma(whd::lanes_sum_f64<L>(sum), P.per_d, static_cast<double>(P.eps));
      const double r = __builtin_amdgcn_rsq(mean);  // to 2^-22 or so, and Newton's step
      return mean < INFINITY ? r * __builtin_fma(-0.5 * mean * r, r, 1.5) : r;
    };
    if (is_q) {
      if (P.q_norm) {
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < PP; u++)
          if (in[u]) sum = __builtin_fmaf(x[n][u], x[n][u], __builtin_fmaf(y[n][u], y[n][u], sum));
        const float mean = __builtin_fmaf(lanes_sum<L>(sum), static_cast<float>(P.per_d), P.eps);
        const bool apart = !(mean >= 0x1p-126f && mean < INFINITY);  // not f32's: values beyond 2^-63 .. 2^63
        if (__builtin_expect(__ballot(apart) == 0, 1)) {
          const float r = __builtin_amdgcn_rsqf(mean);  // off by a unit of f32 at most
#pragma unroll
          for (int u = 0; u < PP; u++) x[n][u] = x[n][u] * r * qw[u][0], y[n][u] = y[n][u] * r * qw[u][1];
        } else {
          const double r = root64();
#pragma unroll
          for (int u = 0; u < PP; u++)
            x[n][u] = static_cast<float>(x[n][u] * r * qw[u][0]), y[n][u] = static_cast<float>(y[n][u] * r * qw[u][1]);
        }
      }
    } else {
      const double r = P.k_norm ? root64() : 1.0;
#pragma unroll
      for (int u = 0; u < PP; u++) {
        const double nx = x[n][u] * r * kw[u][0], ny = y[n][u] * r * kw[u][1];
        kx[u] = turned[u] ? nx * cs[u] - ny * sn[u] : nx;
        ky[u] = turned[u] ? nx * sn[u] + ny * cs[u] : ny;
      }
    }
    if (h >= n_slots) continue;
#pragma unroll
    for (int u = 0; u < PP; u++) {
      if (!in[u]) continue;
      if (is_q) {
        if (P.q_out) {
          const float c = static_cast<float>(cs[u]), s = static_cast<float>(sn[u]);
          float* o = P.q_out + row * P.ldq_out + static_cast<size_t>(h) * P.d;
          const float other = present ? __builtin_nanf("") : 0.f;
          const float ox = turned[u] ? x[n][u] * c - y[n][u] * s : x[n][u], oy = turned[u] ? x[n][u] * s + y[n][u] * c : y[n][u];
          o[a[u]] = present && fits ? ox : other;
          o[b[u]] = present && fits ? oy : other;
        }
      } else {
        const uint32_t kh = h - P.n_heads;
        if (P.k_out) {
          float* o = P.k_out + row * P.ldk_out + static_cast<size_t>(kh) * P.d;
          o[a[u]] = present ? static_cast<float>(kx[u]) : 0.f;
          o[b[u]] = present ? static_cast<float>(ky[u]) : 0.f;
        }
        if (P.k_cache && present && fits) {
          const size_t at = ((m * P.max_rows + static_cast<size_t>(i)) * P.n_kv + kh) * P.d;
          P.k_cache[at + a[u]] = stored(kx[u]);
          P.k_cache[at + b[u]] = stored(ky[u]);
          P.v_cache[at + a[u]] = static_cast<_Float16>(vx[n][u]);
          P.v_cache[at + b[u]] = static_cast<_Float16>(vy[n][u]);
        }
      }
    }
  }
}

template <int L, int PP>
int launch(const Params& P, hipStream_t s) {
  const uint32_t slots = P.n_heads + P.n_kv;
  Params A = P;
  // Few rows: the launch is as long as its dependent loads, and takes as many waves as there are
  // pairs of heads; many rows: a wave's heads share the angles.  Rows of 32 / 8 heads of 128 with
  // 2 and 4 heads to a wave: 60 rows 3.4, 3.6 us, 150 4.2, 4.2, 300 6.1, 5.6, 1200 14.6, 11.8; 4000
  // with 4, 5, 8 and 10 heads 35.5, 35.9, 35.5, 35.2, in neighbouring pairs 37.3, 40.8, 38.4, 38.1,
  // normed 41.7, 42.0, 41.2, 41.1.  Wider heads gain nothing from it (16 / 4 heads of 256 with 2, 3,
  // 4 and 5: 2000 rows 24.6, 25.0, 27.0, 25.6, 4000 42.4, 41.7, 45.1, 43.7; 32 / 8 of 160, 4000
  // rows: 65.9, 65.5, 64.6, 71.2).
  const bool many = PP == 1 && static_cast<size_t>(P.rows) * slots >= kManyHeads;
  const uint32_t per = 64 / L * (many ? 4 : 2);
  A.groups = (slots + per - 1) / per;
  const size_t items = static_cast<size_t>(P.rows) * A.groups;
  const size_t workgroups = (items + kThreads / 64 - 1) / (kThreads / 64), x = workgroups < kGridWidth ? workgroups : kGridWidth;
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>((workgroups + x - 1) / x));  // items below 2^31: at most 2^7 rows
  if constexpr (PP == 1) {
    if (many) rope_kernel<L, PP, 4><<<grid, kThreads, 0, s>>>(A);
    else rope_kernel<L, PP, 2><<<grid, kThreads, 0, s>>>(A);
  } else {
    rope_kernel<L, PP, 2><<<grid, kThreads, 0, s>>>(A);
  }
  WH_LAUNCH_CHECK("norm and rotation launch");
  return WH_OK;
}

}  // namespace

namespace wh {

int check_rope_rules(const char* fn, const wh_rope_rules& r, size_t head_dim) {
  if (head_dim == 0 || head_dim % 2 != 0 || head_dim > 256)
    return set_error(WH_ERR_INVALID_SHAPE, "%s: head_dim %zu is not an even number up to 256", fn, head_dim);
  if (r.rot_dim % 2 != 0 || r.rot_dim > head_dim)
    return set_error(WH_ERR_INVALID_SHAPE, "%s: rot_dim %zu is not an even number up to head_dim %zu", fn, r.rot_dim, head_dim);
  if (!r.inv_freq) return set_error(WH_ERR_INVALID_ARGUMENT, "%s: null inv_freq", fn);
  if (!aligned(r.inv_freq, 4) || !aligned(r.q_norm, 4) || !aligned(r.k_norm, 4))
    return set_error(WH_ERR_INVALID_ARGUMENT, "%s: inverse frequencies and norm weights must be 4-byte aligned", fn);
  if (!(r.magnitude - r.magnitude == 0.0)) return set_error(WH_ERR_INVALID_ARGUMENT, "%s: the magnitude must be finite", fn);
  if ((r.q_norm || r.k_norm) && !(r.norm_eps >= 0.f && r.norm_eps <= 3.402823466e38f))
    return set_error(WH_ERR_INVALID_ARGUMENT, "%s: norm_eps must be finite and not below 0", fn);
  return WH_OK;
}

int launch_rope(const wh_rope_rules& r, const RopeArgs& a, hipStream_t s) {
  Params P{};
  P.q = a.q, P.k = a.k, P.v = a.v;
  P.ldq = a.ldq, P.ldkv = a.ldkv, P.ldq_out = a.ldq_out, P.ldk_out = a.ldk_out;
  P.max_rows = a.max_rows;
  P.base_len = a.base_len, P.len = a.len;
  P.inv_freq = r.inv_freq, P.q_norm = r.q_norm, P.k_norm = r.k_norm;
  P.q_out = a.q_out, P.k_out = a.k_out;
  P.k_cache = static_cast<_Float16*>(a.k_cache), P.v_cache = static_cast<_Float16*>(a.v_cache);
  P.n_per = static_cast<uint32_t>(a.n_per), P.n_new = static_cast<uint32_t>(a.n_new);
  P.n_heads = static_cast<uint32_t>(a.n_heads), P.n_kv = static_cast<uint32_t>(a.n_kv_heads);
  P.d = static_cast<uint32_t>(a.head_dim);
  P.half = static_cast<uint32_t>((r.rot_dim ? r.rot_dim : a.head_dim) / 2);
  P.rows = static_cast<uint32_t>(a.n_members * a.n_new);
  P.interleaved = r.interleaved;
  P.eps = r.norm_eps;
  P.per_d = 1.0 / static_cast<double>(a.head_dim);
  P.magnitude = r.magnitude == 0.0 ? 1.0 : r.magnitude;
  return P.d <= 64 ? launch<32, 1>(P, s) : P.d <= 128 ? launch<64, 1>(P, s) : launch<64, 2>(P, s);
}

}  // namespace wh

WH_API int wh_rope_scaled_inv_freq(int kind, float base, size_t rot_dim, float factor, size_t original_ctx, float low,
                                   float high, float* out_host, double* magnitude) {
  const char* const fn = "rope_scaled_inv_freq";
  if (kind < WH_ROPE_PLAIN || kind > WH_ROPE_BY_INDEX)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: unknown kind %d", fn, kind);
  if (!out_host) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null output", fn);
  if (rot_dim == 0 || rot_dim % 2 != 0 || (kind == WH_ROPE_BASE && rot_dim == 2))
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: rot_dim %zu must be even, and above 2 for a scaled base", fn, rot_dim);
  const bool ramp = kind == WH_ROPE_BY_TURNS || kind == WH_ROPE_BY_INDEX;
  const float most = 3.402823466e38f;
  if (!(base > 0.f && base <= most) || (kind == WH_ROPE_BY_INDEX && !(base > 1.f)))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: the base must be finite and above 0 (1 for steps of the index)", fn);
  if (kind != WH_ROPE_PLAIN && !(factor > 0.f && factor <= most))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: the factor must be finite and above 0", fn);
  if (ramp && (original_ctx == 0 || !(low > 0.f && low < high && high <= most)))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: the kind needs original_ctx and 0 < low < high", fn);
  const double d = static_cast<double>(rot_dim), two_pi = 6.283185307179586, ctx = static_cast<double>(original_ctx);
  const double b = kind == WH_ROPE_BASE ? base * pow(static_cast<double>(factor), d / (d - 2.0)) : static_cast<double>(base);
  // the index whose frequency makes `turns` turns within the context
  auto index_of = [&](double turns) { return d * log(ctx / (turns * two_pi)) / (2.0 * log(b)); };
  double first = 0.0, last = 0.0;
  if (kind == WH_ROPE_BY_INDEX) {  // bounds and step of the published YaRN method, by which models are trained
    first = fmax(floor(index_of(high)), 0.0);
    last = fmin(ceil(index_of(low)), d - 1.0);
    if (!(last > first)) last = first + 0.001;  // a step
  }
  for (size_t i = 0; i < rot_dim / 2; i++) {
    const double f = 1.0 / pow(b, 2.0 * static_cast<double>(i) / d);
    double g = kind == WH_ROPE_LINEAR ? 0.0 : 1.0;
    if (kind == WH_ROPE_BY_TURNS) g = (ctx * f / two_pi - low) / (static_cast<double>(high) - low);
    if (kind == WH_ROPE_BY_INDEX) g = 1.0 - (static_cast<double>(i) - first) / (last - first);
    g = fmin(fmax(g, 0.0), 1.0);
    const double by = kind == WH_ROPE_PLAIN || kind == WH_ROPE_BASE ? 1.0 : static_cast<double>(factor);
    out_host[i] = static_cast<float>(f * (g + (1.0 - g) / by));
  }
  if (magnitude)
    *magnitude = kind == WH_ROPE_BY_INDEX && factor > 1.f ? 0.1 * log(static_cast<double>(factor)) + 1.0 : 1.0;
  return WH_OK;
}

WH_API int wh_qk_norm_rope(const wh_rope_rules* rules, const float* q, const float* k, const float* v, size_t ldq,
                           size_t ldkv, const uint32_t* base_len, const uint32_t* len, size_t n_groups, size_t n_per,
                           size_t n_new, size_t n_heads, size_t n_kv_heads, size_t head_dim, float* q_out, size_t ldq_out,
                           float* k_out, size_t ldk_out, void* k_cache, void* v_cache, size_t max_rows,
                           wh_stream_t stream) {
  const char* const fn = "qk_norm_rope";
  if (!rules) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null rules", fn);
  const int st = wh::check_rope_rules(fn, *rules, head_dim);
  if (st) return st;
  if (n_heads == 0 || n_kv_heads == 0 || n_heads >> 16 || n_kv_heads >> 16)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: %zu heads, %zu KV heads (1 to 65535)", fn, n_heads, n_kv_heads);
  size_t members, rows, all;
  if (__builtin_mul_overflow(n_groups, n_per, &members) || __builtin_mul_overflow(members, n_new, &rows) ||
      __builtin_mul_overflow(rows, n_heads + n_kv_heads, &all) || all >> 31)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: %zu x %zu members, %zu tokens, %zu heads (together fewer than 2^31)", fn,
                         n_groups, n_per, n_new, n_heads + n_kv_heads);
  const size_t qd = n_heads * head_dim, kvd = n_kv_heads * head_dim;
  if (ldq < qd || ldkv < kvd || (q_out && ldq_out < qd) || (k_out && ldk_out < kvd))
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: row strides %zu, %zu, %zu, %zu below the rows' %zu and %zu elements", fn, ldq,
                         ldkv, ldq_out, ldk_out, qd, kvd);
  if ((k_cache != nullptr) != (v_cache != nullptr))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: one cache without the other", fn);
  if (k_cache && (max_rows == 0 || max_rows >> 31))
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: max_rows = %zu out of range", fn, max_rows);
  if (rows == 0) return WH_OK;
  if (!q || !k || (k_cache && !v)) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  const void* ptrs[] = {q, k, v, base_len, len, q_out, k_out};
  for (const void* p : ptrs)
    if (!wh::aligned(p, 4)) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: arrays must be 4-byte aligned", fn);
  if (!wh::aligned(k_cache, 2) || !wh::aligned(v_cache, 2) || (k_cache && k_cache == v_cache))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: caches must be 2-byte aligned, and two", fn);
  if ((q_out == q && ldq_out != ldq && q_out) || (k_out == k && ldk_out != ldkv && k_out))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: in place, both strides must be the same", fn);
  if (!q_out && !k_out && !k_cache) return WH_OK;
  const wh::RopeArgs a{q,          k,        v,     ldq,     ldkv,  base_len, len,     members, n_per,   n_new, n_heads,
                       n_kv_heads, head_dim, q_out, ldq_out, k_out, ldk_out,  k_cache, v_cache, max_rows};
  return wh::launch_rope(*rules, a, reinterpret_cast<hipStream_t>(stream));
}
