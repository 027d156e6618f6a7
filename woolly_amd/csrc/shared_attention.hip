// shared_attention.hip -- grouped-query attention of one query per member over
// cache rows that its group shares (the prefix) and rows of its own, on gfx950.
//
// With G = n_heads / n_kv_heads and n_per members to a group:
//   s_j = (q . k_j) / sqrt(d) over the prefix's and the member's own rows
//   out = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},  m = max_j s_j
// The prefix's rows are read once for the n_per G query rows that a KV head has
// in a group.  Two launches:
//   1. partial: a workgroup per (KV head, 32, 64 or 128 query rows, chunk of the
//      prefix), and per (KV head, member, chunk of its own rows): maximum, sum and
//      weighted sum of V of each row
//   2. combine: a wave, or four, per 32 query rows and 8 dims join their chunks
// The chunks' number is the launch's, their length follows from the lengths on
// the device.
//
// Products on the matrix cores (v_mfma_f32_32x32x16_f16), as tree_attention.hip
// has them: S^T = K Q^T leaves a lane with 16 keys of one query row, in the order
// in which the registers are the B operand of O^T = V^T P^T.  q, scaled by a power
// of two, and the weights are split into two f16 limbs each, K and V are taken as
// they are.  A weight is 2^12 e^{s - m}, m a reference that follows the tiles' largest
// scores up and down, its low limb held times 2^11 and summed apart in each tile: it
// keeps 2^-22 of itself down to 2^-26 of the reference's, and 2^-48 of that below.
// Beside one key with nearly all the weight (often the first one, whose v is small) the
// others make the output, and keep what f32 would leave them: m moves down to them, and
// that key's own tile takes two turns.  Relative L2 with 90 to 99.9999999 % on one key of
// 60000: 2e-7 to 4e-6 (with m the running maximum alone up to 2e-2).  Calls whose scores have a
// deviation up to 5 take what they took with that: 48 members at 131000 253 -> 251 us, 64 at 20000
// 63 -> 62, 32 at 60000 of 64 dims 49.5 -> 48.5, 8 at 30000 33.7 -> 33.8, 4 at 900 10.2 -> 10.5; with 8
// the first takes 300, with 16 435, where most tiles have keys far apart.  Moving up, which the
// first tiles do, in one block with the rest cost another 1 to 3 %.
//
// Few query rows: a wave has its own tiles of 32 keys, its own LDS and no barriers
// until the chunk's end; memory bounds it (8 members at 30000 + 250 rows, 131 MB,
// 34 us with both launches).  Many: the waves share stages of 64 keys; bound by matrix and
// vector instructions that take turns, under a clock that falls with such work: 48 members at
// 131000 + 400 rows, 206 GFLOP of limbs, 255 us; of a SIMD's cycles 42 % are the matrix
// cores' and 45 % vector instructions', and a wave has its scores, weights and values one
// behind the other, with a branch between scores and weights across which nothing moves.
// The places are cut for max_prefix and max_own: in a cache of 131072 rows 64 members at
// 6000 take 36 us instead of 31, 4 at 900 12.7 instead of 10.4.
#include <type_traits>

#include "attn_dev.hpp"
#include "members.hpp"
#include "tree.hpp"

namespace {

using whd::f32x16, whd::f32x4u, whd::s16x4;
using whd::read_tr, whd::swap_max, whd::swap_max_nan, whd::swap_sum, whd::swz_k, whd::swz_v;

constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
// Weights are held in f16 as 2^12 e^{s - m}.  The reference m of a row moves up to a tile's largest
// score where that is above 2^3 of it (at most 2^15 in f16), and down to it, but never 2^48 below its
// highest, where it is faint: below 2^-30 (2^-18 in f16, where the low limb is off by 2^-18 of it).
// A tile with a key far above its neighbours takes two turns: the keys down to 2^-9 of it, then the
// others.  Half of a row's keys in a tile are one lane's, and such a key is told by the other half,
// faint against it, and by being within 2^-10 of the row's highest.  (Such keys in both halves
// hide the rest of their tile.)  Of 32 rows with scores of deviation 1.3, 3 and 5 some row's m moves
// up in 10, 12 and 16 % of the tiles, none down; with 8 it is 50 % and 9 %, and 2 % take two turns; with
// 16 all, 83 and 50 %.
constexpr float kPScaleLog2 = 12.0f, kMoveUp = 3.0f, kLowest = 48.0f;
constexpr float kFaint = -30.0f, kNear = -9.0f, kHigh = -10.0f;
constexpr float kLowScale = 0x1p11f, kLowUnscale = 0x1p-11f;
constexpr uint32_t kLeastChunk = 128;  // keys: a tile for every wave
constexpr double kShareFrom = 10.0;    // work (plan)
constexpr uint32_t kStageKeys = 64;    // of a workgroup of 128 query rows
// LDS reads run one step ahead of the matrix products that take them: neither moves
// across this
constexpr int kNoLds = 0x406;

struct Params {
  const float* q;
  size_t ldq;
  const uint32_t *prefix_len, *own_len;
  const _Float16 *k_prefix, *v_prefix, *k_own, *v_own;
  float* out;
  uint32_t n_groups, n_per, max_prefix, max_own, n_heads, n_kv, G;
  uint32_t R;            // query rows of a KV head in a group: n_per G
  uint32_t tiles;        // of 32 of them
  uint32_t own_tiles;    // of a member's G
  uint32_t own_rows;     // rows of such a tile that are stored: min(G, 32)
  uint32_t cp, co;       // chunks of a prefix, of a member's own rows
  uint32_t slots;        // chunks of all prefixes: cp each, or (shared) as the lengths are
  int shared, sorted;    // sorted: members with the longest own rows first
  uint32_t n_prefix_wgs;
  uint32_t rw;           // tiles of a prefix's workgroup
  float scale;           // log2(e) / sqrt(d)
  // workspace: partial results (largest score of the row in units of q . k, sum), registers
  // of the lanes [D / 8][2][rows]
  float2* ml_p;          // [slots][n_kv][tiles][32]
  float4* acc_p;
  float2* ml_o;          // [members][co][n_kv][own_tiles][own_rows]
  float4* acc_o;
};

// Cache rows of a group's prefix and of a member, 0 where they do not fit.
__device__ __forceinline__ uint32_t rows_of(const uint32_t* len, uint32_t i, uint32_t most) {
  const uint32_t n = len ? len[i] : 0;
  return n <= most ? n : 0;
}
__device__ __forceinline__ uint32_t chunk_of(uint32_t rows, uint32_t chunks) {
  const uint32_t even = (rows + chunks - 1) / chunks;
  return max((even + kLeastChunk - 1) / kLeastChunk * kLeastChunk, kLeastChunk);
}

// Groups whose prefixes differ in length share the slots: about the shortest chunks that fit
// into them.  Lane l has group l.  With n = ceil(units / per) in
// f32: a quotient is off by 2^-22 of itself and, below 2^20 units, an integer or at least 2^-20
// of itself above one.
struct Shares {
  uint32_t rows, n, upto;  // of the lane's group: cache rows, chunks, chunks up to its last one
  uint32_t chunk;
};
__device__ __forceinline__ uint32_t lane_of(uint32_t v, uint32_t lane) {
  return __builtin_amdgcn_readlane(v, __builtin_amdgcn_readfirstlane(lane));
}
__device__ __forceinline__ Shares shares_of(const Params& P, uint32_t lane) {
  Shares a;
  a.rows = lane < P.n_groups ? rows_of(P.prefix_len, lane, P.max_prefix) : 0;
  const uint32_t units = (a.rows + kLeastChunk - 1) / kLeastChunk;
  const uint32_t all = whd::wave_join(units, [](uint32_t x, uint32_t y) { return x + y; });
  auto quotient = [](uint32_t u, uint32_t by) {
    return ceilf(static_cast<float>(u) * (__builtin_amdgcn_rcpf(static_cast<float>(by)) * (1.f - 0x1p-21f)));
  };
  // of chunks of `least` units there may be too many, of `most` there are not: each group rounds up once
  uint32_t least = max((all + P.slots - 1) / P.slots, 1u), most = max((all + P.slots - P.n_groups - 1) / (P.slots - P.n_groups), 1u);
  auto fits = [&](uint32_t per) {
    return whd::wave_join(static_cast<uint32_t>(quotient(units, per)), [](uint32_t x, uint32_t y) { return x + y; }) <= P.slots;
  };
  if (fits(least)) most = least;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t mid = least + (most - least) / 2;
    if (fits(mid)) most = mid; else least = mid;
  }
  const uint32_t per = __builtin_amdgcn_readfirstlane(most);
  a.chunk = per * kLeastChunk;
  a.n = static_cast<uint32_t>(quotient(units, per));
  // sums over the lanes up to this one: within rows of 16, then the rows before
  uint32_t v = a.n;
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x111, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x112, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x114, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x118, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x142, 0xA, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x143, 0xC, 0xF, false));
  a.upto = v;
  return a;
}

// The i-th of up to 64 members with the longest own rows first (to an eighth of the longest).
__device__ __forceinline__ uint32_t by_length(const Params& P, uint32_t i, uint32_t lane) {
  const bool here = lane < P.n_groups * P.n_per;
  const uint32_t rows = here ? rows_of(P.own_len, lane, P.max_own) : 0;
  const uint32_t most = whd::wave_join(rows, [](uint32_t x, uint32_t y) { return max(x, y); });
  const int eighth = here ? static_cast<int>(static_cast<float>(rows) * (7.99f * __builtin_amdgcn_rcpf(static_cast<float>(max(most, 1u))))) : -1;
  uint32_t place = 0, before = 0;
#pragma unroll
  for (int e = 7; e >= 0; e--) {
    const unsigned long long those = __ballot(eighth == e);
    if (eighth == e) place = before + __builtin_popcountll(those & ((1ull << lane) - 1));
    before += __builtin_popcountll(those);
  }
  return __builtin_ctzll(__ballot(here && place == i));
}

// Two weights as f16 hi + lo 2^-11: elements i and i + 1 of the fragments.
__device__ __forceinline__ void split2(float a, float b, half8& hi, half8& lo, int i) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const half2v h = __builtin_convertvector((f32x2{a, b}), half2v);
  const uint32_t hw = __builtin_bit_cast(uint32_t, h);
  float ra, rb;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hw), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hw), "v"(b));
  const half2v r = __builtin_convertvector((f32x2{ra * kLowScale, rb * kLowScale}), half2v);
  hi[i] = h[0], hi[i + 1] = h[1];
  lo[i] = r[0], lo[i + 1] = r[1];
}

template <int D>
struct Shape {
  static constexpr int KS = D / 16, DT = D / 32, kQuads = D / 8;
  static constexpr int kTile = 32 * D * 2;       // bytes of 32 rows of K or V
  static constexpr int kCopies = kTile / 1024;   // copies of 1 KB per tile
  static constexpr int kPer = 1024 / (2 * D);    // rows of a copy
  static constexpr int kStage = kWaves * 2 * kTile;
  static constexpr int kMerge = kWaves * 32 * (D + 2) * 4;
  static constexpr int kLds = kStage > kMerge ? kStage : kMerge;
};

// The query rows of a wave and what it has summed over its keys.
template <int D>
struct Rows {
  half8 qh[D / 16], ql[D / 16];
  float qs;  // log2(e) / sqrt(d) of a product of scaled q and k
  int e;     // q is scaled by 2^e
  f32x16 acc[D / 32];
  float m, l;
  float peak;  // m before it last went down, or the highest of those
};

// q rows: lane l has row l % 32, elements 16 j + 8 (l / 32) .. of each step j.
template <int D>
__device__ __forceinline__ void load_rows(Rows<D>& w, const float* q, float scale, int h) {
  constexpr int KS = D / 16;
  float x[KS][8];
#pragma unroll
  for (int j = 0; j < KS; j++) {
    const f32x4u a = *reinterpret_cast<const f32x4u*>(q + 16 * j + 8 * h), b = *reinterpret_cast<const f32x4u*>(q + 16 * j + 8 * h + 4);
#pragma unroll
    for (int u = 0; u < 4; u++) x[j][u] = a[u], x[j][4 + u] = b[u];
  }
  float mx = 0.f;
#pragma unroll
  for (int j = 0; j < KS; j++)
#pragma unroll
    for (int u = 0; u < 8; u++) mx = fmaxf(mx, fabsf(x[j][u]));
  mx = swap_max(mx);
  // the row's largest magnitude to [2^13, 2^14): hi + lo hold every element to 2^-22 of
  // itself or 2^-38 of the largest
  w.e = mx > 0.f && mx < INFINITY ? min(13 - ilogbf(mx), 100) : 0;
#pragma unroll
  for (int j = 0; j < KS; j++)
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const float v = ldexpf(x[j][u], w.e);
      const _Float16 hi = static_cast<_Float16>(v);
      w.qh[j][u] = hi;
      w.ql[j][u] = static_cast<_Float16>(v - static_cast<float>(hi));
    }
  w.qs = ldexpf(scale, -w.e);
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) w.acc[d][i] = 0.f;
  w.m = w.peak = -INFINITY;
  w.l = 0.f;
}

// The operands of the 32 keys of the K tile at kt (LDS), 16 elements of their rows to a step.
template <int D>
struct Keys {
  uint32_t at;
  __device__ __forceinline__ Keys(uint32_t kt, int l32, int h) : at(kt + l32 * 2 * D + 16 * (h ^ swz_k<D>(l32))) {
    asm("" : "+v"(at));  // the steps' addresses are made of it each time: they would take registers across the loop
  }
  __device__ __forceinline__ half8 step(int j) const {
    return *reinterpret_cast<const __attribute__((address_space(3))) half8*>((uintptr_t)(at ^ (32 * j)));
  }
};

// Scores of the keys, key 8 (i / 4) + 4 h + i % 4 in s[i].
template <int D>
__device__ __forceinline__ void scores(const Rows<D>& w, const Keys<D>& keys, f32x16& s) {
  constexpr int KS = D / 16;
#pragma unroll
  for (int i = 0; i < 16; i++) s[i] = 0.f;
  half8 k[2];
  k[0] = keys.step(0);
#pragma unroll
  for (int j = 0; j < KS; j++) {
    if (j + 1 < KS) k[(j + 1) & 1] = keys.step(j + 1);
    __builtin_amdgcn_sched_barrier(kNoLds);
    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[j & 1], w.qh[j], s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[j & 1], w.ql[j], s, 0, 0, 0);
  }
}

// A score that is NaN: the formula's, or made of an infinity in K that q's limbs meet with
// both signs or as 0.  q's sign and size are the hi limb's: its product alone says what an
// infinity makes of the score.
template <int D>
__device__ __forceinline__ void mend_scores(const Rows<D>& w, const Keys<D>& keys, f32x16& s) {
  constexpr int KS = D / 16;
  f32x16 x;
#pragma unroll
  for (int i = 0; i < 16; i++) x[i] = 0.f;
#pragma unroll 1
  for (int j = 0; j < KS; j++) {
    half8 q = w.qh[0];
#pragma unroll
    for (int u = 1; u < KS; u++) q = j == u ? w.qh[u] : q;
    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys.step(j), q, x, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (s[i] != s[i]) s[i] = x[i];
}

// Brings the row's reference, and with it the sums so far, to the scores of N tiles.  Returns
// whether the tiles need a second turn, for the keys that it has left out of this one.
// mend: mend_scores of the tiles.
template <int D, int N, bool SECOND, typename Mend>
__device__ __forceinline__ bool settle(Rows<D>& w, f32x16 (&s)[N], std::bool_constant<SECOND>, const Mend& mend) {
  float top, mt;  // the largest score of the lane's half, and of the row; NaN if there is one
  auto largest = [&]() __attribute__((always_inline)) {
    top = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * N; i++) top = __builtin_elementwise_maximum(top, s[i / 16][i % 16]);
    mt = swap_max_nan(top);
  };
  largest();
  auto move = [&](bool moves, float to) __attribute__((always_inline)) {
    const float al = moves ? __builtin_amdgcn_exp2f((w.m - to) * w.qs) : 1.f;
    w.l *= al;
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) w.acc[d][i] *= al;
    if (moves) w.m = to;
  };
  auto mend_nan = [&]() __attribute__((always_inline)) {
    if (__builtin_expect(__ballot(mt != mt) == 0, 1)) return;
    mend();
    largest();  // NaN still: the row is NaN
  };
  if constexpr (SECOND) {
    mend_nan();
  } else {
    if (__ballot(!((mt - w.m) * w.qs <= kMoveUp))) {  // NaN comes here
      mend_nan();
      move(!((mt - w.m) * w.qs <= kMoveUp) && mt != -INFINITY, mt);
    }
    if (__builtin_expect(__ballot((top - w.m) * w.qs < kFaint) == 0, 1)) return false;
  }
  // What is faint counts down to 2^-78 of the row's highest, where m cannot follow.
  const float unit = __builtin_amdgcn_rcpf(w.qs);
  w.peak = fmaxf(w.peak, w.m);
  auto counts = [&](float score, float ref) { return (score - ref) * w.qs < kFaint && (score - w.peak) * w.qs >= kFaint - kLowest; };
  bool again = false;
  if (SECOND || __ballot((mt - w.peak) * w.qs >= kHigh && counts(top, mt))) {
    const float split = __builtin_fmaf(kNear, unit, mt);
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[n][i] = (s[n][i] < split) != SECOND ? -INFINITY : s[n][i];
    float most = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * N; i++) most = fmaxf(most, s[i / 16][i % 16]);
    mt = swap_max(most);
    again = !SECOND;
  }
  move(counts(mt, w.m), fmaxf(mt, w.peak - kLowest * unit));
  return again;
}

// The weights of the scores of N tiles, as hi and lo limbs.
template <int D, int N>
__device__ __forceinline__ void weigh(Rows<D>& w, const f32x16 (&s)[N], half8 (&ph)[2 * N], half8 (&pl)[2 * N]) {
  const float mb = w.m == -INFINITY ? 0.f : w.m;
  float lt[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < 2 * N; ks++)
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float p[2];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        p[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks / 2][8 * (ks % 2) + i + k] - mb, w.qs, kPScaleLog2));
        lt[(i + k) & 3] += p[k];
      }
      split2(p[0], p[1], ph[ks], pl[ks], i);
    }
  w.l += (lt[0] + lt[1]) + (lt[2] + lt[3]);
}

// acc += V^T P^T of N V tiles, one behind the other from vt on.
template <int D, int N>
__device__ __forceinline__ void add_values(Rows<D>& w, uint32_t vt, const half8 (&ph)[2 * N], const half8 (&pl)[2 * N], int lane) {
  const int h = lane >> 5, kq = (lane & 15) >> 2, dq = lane & 3, dg = (lane >> 4) & 1;
  uint32_t vo = vt + (4 * h + kq) * 2 * D + 16 * ((2 * dg + (dq >> 1)) ^ swz_v<D>(kq)) + 8 * (dq & 1);
  asm("" : "+v"(vo));
  constexpr int kSteps = D / 32 * 2 * N;
  auto v_at = [&](int step) {  // 32 dims step / (2 N), 16 keys step % (2 N)
    const int d = step / (2 * N), ks = step % (2 * N);
    half8 v;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const s16x4 x = read_tr((vo ^ (64 * d)) + (16 * ks + 8 * u) * 2 * D);
      const auto y = __builtin_bit_cast(_Float16 __attribute__((ext_vector_type(4))), x);
#pragma unroll
      for (int i = 0; i < 4; i++) v[4 * u + i] = y[i];
    }
    return v;
  };
  half8 v[2];
  v[0] = v_at(0);
#pragma unroll
  for (int d = 0; d < D / 32; d++) {
    f32x16 t;
#pragma unroll
    for (int i = 0; i < 16; i++) t[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 2 * N; ks++) {
      const int step = d * 2 * N + ks;
      if (step + 1 < kSteps) v[(step + 1) & 1] = v_at(step + 1);
      __builtin_amdgcn_sched_barrier(kNoLds);
      t = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[step & 1], pl[ks], t, 0, 0, 0);
      w.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[step & 1], ph[ks], w.acc[d], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) w.acc[d][i] = __builtin_fmaf(t[i], kLowUnscale, w.acc[d][i]);
  }
}

// Keys from `left` on of a tile are not there: their scores are -inf, their rows of V
// cleared (they repeat the last row, and 0 times an infinity would be NaN).
__device__ __forceinline__ void mask_scores(f32x16& s, int left, int h) {
#pragma unroll
  for (int i = 0; i < 16; i++) s[i] = 8 * (i >> 2) + 4 * h + (i & 3) < left ? s[i] : -INFINITY;
}
template <int D>
__device__ __forceinline__ void clear_values(uint32_t vt, int left, int lane) {
  constexpr int kPer = 1024 / (2 * D);
  const int row = lane / (D / 8);
  for (int j = max(left, 0) / kPer; j < 32 / kPer; j++)
    if (row + kPer * j >= left)
      *reinterpret_cast<__attribute__((address_space(3))) u32x4*>((uintptr_t)(vt + 1024 * j + 16 * lane)) = u32x4{0, 0, 0, 0};
}

// Infinities and NaN of V: limbs and a weight's 0 make NaN of them.  A weight is above 0,
// however small, but for a score of -inf, so such an element's sum is that of the infinities
// and NaN alone, or NaN (0 times infinity): the rows are read again for them.  Keys
// c0 + 32 first .. in steps of `step` tiles.
template <int D>
__device__ __forceinline__ void mend_values(Rows<D>& w, const uint8_t* kbase, const uint8_t* vbase, size_t RS, uint32_t c0, uint32_t c1,
                                            uint32_t first, uint32_t step, int lane) {
  float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) zero[i & 3] = __builtin_fmaf(w.acc[d][i], 0.f, zero[i & 3]);
  if (__builtin_expect(__ballot(!((zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.f)) == 0, 1)) return;
  const int h = lane >> 5;
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int i = 0; i < 16; i++)
      if (!(fabsf(w.acc[d][i]) < INFINITY)) w.acc[d][i] = 0.f;
  for (uint32_t base = c0 + 32 * first; base < c1; base += 32 * step) {
    const uint32_t look = min(base + lane / 2, c1 - 1);  // lane l looks through half of row l / 2
    const uint4* half = reinterpret_cast<const uint4*>(vbase + look * RS + (lane & 1) * D);
    bool bad = false;
    for (int j = 0; j < D / 16; j++) {
      const uint4 x4 = half[j];
      for (const uint32_t x : {x4.x, x4.y, x4.z, x4.w}) bad |= (x & 0x7C00u) == 0x7C00u || (x & 0x7C000000u) == 0x7C000000u;
    }
    unsigned long long rows_bad = __ballot(bad);
    rows_bad = (rows_bad | rows_bad >> 1) & 0x5555555555555555ull;  // bit 2 k: row k
    while (rows_bad) {
      const uint32_t key = base + __builtin_ctzll(rows_bad) / 2;
      rows_bad &= rows_bad - 1;
      if (key >= c1) break;  // the last row, looked at again
      const _Float16 *k = reinterpret_cast<const _Float16*>(kbase + key * RS), *v = reinterpret_cast<const _Float16*>(vbase + key * RS);
      float score = 0.f;  // -inf as mend_scores has it
#pragma unroll
      for (int j = 0; j < D / 16; j++) {
        u32x4 q = __builtin_bit_cast(u32x4, w.qh[j]);
        asm volatile("" : "+v"(q)::"memory");  // a step at a time: this is rare, and short of registers
        const half8 a = *reinterpret_cast<const half8*>(k + 16 * j + 8 * h), b = __builtin_bit_cast(half8, q);
#pragma unroll
        for (int u = 0; u < 8; u++) score = __builtin_fmaf(static_cast<float>(a[u]), static_cast<float>(b[u]), score);
      }
      const bool none = swap_sum(score) == -INFINITY;
#pragma unroll
      for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float x = static_cast<float>(v[32 * d + 8 * (i >> 2) + 4 * h + (i & 3)]);
          if (!(fabsf(x) < INFINITY)) w.acc[d][i] += none ? __builtin_nanf("") : x;
        }
    }
  }
}

// What a workgroup works on.
struct Work {
  const uint8_t *k, *v;   // row 0 of its KV head
  uint32_t c0, c1;        // its keys
  uint32_t member0;       // query row r: member member0 + r / G, head kvh G + r % G
  uint32_t row0, n_rows;  // its first query row, and how many there are
  uint32_t kvh;
  float2* ml;             // [stored]
  float4* acc;            // [D / 8][2][stored]
  uint32_t stored;        // rows of a tile that are stored
};

template <int D>
__device__ __forceinline__ void load_rows_of(Rows<D>& w, const Params& P, const Work& W, uint32_t r0, int h) {
  const uint32_t r = min(r0, W.n_rows - 1);
  load_rows(w, P.q + (W.member0 + r / P.G) * P.ldq + static_cast<size_t>(W.kvh * P.G + r % P.G) * D, P.scale, h);
}

// The factor that brings sums to a reference `by` powers of two higher.  Not 0: an infinity stays one.
__device__ __forceinline__ float factor_of(float by) { return __builtin_elementwise_maximum(__builtin_amdgcn_exp2f(by), 0x1p-126f); }

// Waves whose query rows are the same and that have taken keys apart, N of them with
// kWaves / N tiles, join in LDS, in fixed order, and store in the lanes' order.
template <int D, int N>
__device__ __forceinline__ void join_waves(const Rows<D>& w, const Work& W, unsigned char* lds, uint32_t wave, int lane) {
  constexpr int kQuads = D / 8, kApart = kWaves / N;
  const int l32 = lane & 31, h = lane >> 5;
  const uint32_t tile = wave % kApart, part = wave / kApart;
  whd::lds_barrier();
  float4* am = reinterpret_cast<float4*>(lds);                        // [4][D / 8][64]
  float2* mm = reinterpret_cast<float2*>(am + kWaves * kQuads * 64);  // [4][32]
#pragma unroll
  for (int d = 0; d < D / 32; d++)
#pragma unroll
    for (int i = 0; i < 4; i++)
      am[(wave * kQuads + 4 * d + i) * 64 + lane] =
          make_float4(w.acc[d][4 * i], w.acc[d][4 * i + 1], w.acc[d][4 * i + 2], w.acc[d][4 * i + 3]);
  if (h == 0) mm[wave * 32 + l32] = make_float2(w.m, w.l);
  whd::lds_barrier();
  float M = -INFINITY, L = 0.f, ew[N];
  float2 ml[N];
#pragma unroll
  for (int u = 0; u < N; u++) {
    ml[u] = mm[(u * kApart + tile) * 32 + l32];
    M = __builtin_elementwise_maximum(M, ml[u].x);
  }
#pragma unroll
  for (int u = 0; u < N; u++) {
    ew[u] = ml[u].x == -INFINITY ? 0.f : factor_of((ml[u].x - M) * w.qs);
    L = __builtin_fmaf(ml[u].y, ew[u], L);
  }
  if (W.row0 + 32 * tile + l32 >= W.n_rows) return;
  float4* const acc = W.acc + tile * 32 * (D / 4);
#pragma unroll
  for (int q = 0; q < kQuads / N; q++) {
    const int quad = part + N * q;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < N; u++) {
      const float4 a = am[((u * kApart + tile) * kQuads + quad) * 64 + lane];
      A.x = __builtin_fmaf(a.x, ew[u], A.x);
      A.y = __builtin_fmaf(a.y, ew[u], A.y);
      A.z = __builtin_fmaf(a.z, ew[u], A.z);
      A.w = __builtin_fmaf(a.w, ew[u], A.w);
    }
    acc[(quad * 2 + h) * W.stored + l32] = A;
  }
  if (part == 0 && h == 0) W.ml[tile * 32 + l32] = make_float2(ldexpf(M, -w.e), L);
}

// 32 query rows, four waves that share the keys: a wave has tiles wave, wave + 4, ..
// of the chunk, LDS of its own for one K and one V tile, and no barriers until the
// end: the next K tile is asked for when the scores are there, the next V tile when the
// products are.
template <int D>
__device__ __forceinline__ void few_rows(const Params& P, const Work& W, unsigned char* lds) {
  using S = Shape<D>;
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t RS = static_cast<size_t>(P.n_kv) * D * 2;  // bytes between cache rows
  // A tile's rows go to LDS 1 KB at a time: lane l has chunk l % kChunks of row l / kChunks.
  // The chunks' permutation of K alternates between copies, that of V does not.
  constexpr int kChunks = D / 8;
  const uint32_t kt = lds_addr(lds) + wave * 2 * S::kTile, vt = kt + S::kTile;
  const uint32_t crow = lane / kChunks, cchunk = lane % kChunks;
  const uint32_t crs = crow * static_cast<uint32_t>(RS);
  const uint32_t ck = 16 * (cchunk ^ (D == 128 ? crow : crow >> 1)), cv = 16 * (cchunk ^ swz_v<D>(crow));
  constexpr int kTurns = D == 128 ? 4 : 2;  // copies until K's permutation repeats
  auto copy_tile = [&](const uint8_t* src, uint32_t base, uint32_t to, uint32_t chunk, bool is_k) {
    const uint8_t* p = src + base * RS;
    const uint32_t last = W.c1 - 1 - base;
    asm("" : "+v"(chunk));  // made anew each time, as the rows below: across the loop they would take registers
    if (last >= 31) {
#pragma unroll
      for (int j = 0; j < S::kCopies; j++) {
        copy16_to_lds(p, crs + (is_k ? chunk ^ (64 * (j % kTurns)) : chunk), to + 1024 * j);
        p += S::kPer * RS;
      }
    } else {  // rows behind the last one repeat it
      uint32_t row = crow;
#pragma unroll
      for (int j = 0; j < S::kCopies; j++) {
        asm("" : "+v"(row));
        copy16_to_lds(p, min(row, last) * static_cast<uint32_t>(RS) + (is_k ? chunk ^ (64 * (j % kTurns)) : chunk), to + 1024 * j);
        row += S::kPer;
      }
    }
  };
  uint32_t base = W.c0 + 32 * wave;
  const bool any = base < W.c1;
  if (any) {
    copy_tile(W.k, base, kt, ck, true);
    copy_tile(W.v, base, vt, cv, false);
  }
  Rows<D> w;
  load_rows_of(w, P, W, W.row0 + l32, h);
  if (any) {
    wait_vmcnt<0>();
    while (true) {
      const uint32_t next = base + 32 * kWaves, left = W.c1 - base;
      const bool more = next < W.c1;
      auto turn = [&](auto second) __attribute__((always_inline)) {
        f32x16 s[1];
        const Keys<D> keys(kt, l32, h);
        scores(w, keys, s[0]);
        if (left < 32) mask_scores(s[0], left, h);
        const bool again = settle(w, s, second, [&] { mend_scores(w, keys, s[0]); });  // asks what they are: the tile has been read
        if (more && !again) copy_tile(W.k, next, kt, ck, true);
        half8 ph[2], pl[2];
        weigh<D, 1>(w, s, ph, pl);
        if (more && !again) wait_vmcnt<S::kCopies>(); else wait_vmcnt<0>();  // V, not the next K
        if (left < 32) clear_values<D>(vt, left, lane);
        add_values<D, 1>(w, vt, ph, pl, lane);
        return again;
      };
      if (__builtin_expect(turn(std::false_type{}), 0)) turn(std::true_type{});
      if (!more) break;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      copy_tile(W.v, next, vt, cv, false);
      wait_vmcnt<S::kCopies>();  // the next K
      base = next;
    }
    mend_values(w, W.k, W.v, RS, W.c0, W.c1, wave, kWaves, lane);
  }
  w.l = swap_sum(w.l);

  join_waves<D, kWaves>(w, W, lds, wave, lane);
}

// 32 RW query rows, 64 or 128, that share stages of 64 keys in LDS, two of them in
// turn: K and V are read from memory once for all of them.  A wave has 32 rows, of a
// stage all keys or, with 64 rows, half of them.
template <int D, int RW>
__device__ __forceinline__ void many_rows(const Params& P, const Work& W, unsigned char* lds) {
  using S = Shape<D>;
  const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t RS = static_cast<size_t>(P.n_kv) * D * 2;
  constexpr int kChunks = D / 8, kRowsAll = S::kPer * kWaves, kCopies = kStageKeys / kRowsAll;  // the chunks' permutation repeats within kRowsAll rows
  const uint32_t lds0 = lds_addr(lds);
  const uint32_t crow = wave * S::kPer + lane / kChunks, cchunk = lane % kChunks;
  const uint32_t ck = 16 * (cchunk ^ swz_k<D>(crow)), cv = 16 * (cchunk ^ swz_v<D>(crow));
  const uint32_t crs = crow * static_cast<uint32_t>(RS);
  auto issue = [&](uint32_t base, uint32_t buf) {
    const uint8_t *kb = W.k + base * RS, *vb = W.v + base * RS;
    uint32_t at = lds0 + buf * 4 * S::kTile + wave * 1024;
    if (base + kStageKeys <= W.c1) {
#pragma unroll
      for (int j = 0; j < kCopies; j++) {
        copy16_to_lds(kb, crs + ck, at);
        copy16_to_lds(vb, crs + cv, at + 2 * S::kTile);
        kb += kRowsAll * RS;
        vb += kRowsAll * RS;
        at += kWaves * 1024;
      }
    } else {  // rows behind the last one repeat it
      const uint32_t last = W.c1 - 1 - base;
      uint32_t row = crow;
#pragma unroll
      for (int j = 0; j < kCopies; j++) {
        asm("" : "+v"(row));
        const uint32_t at_row = min(row, last) * static_cast<uint32_t>(RS);
        copy16_to_lds(kb, at_row + ck, at);
        copy16_to_lds(vb, at_row + cv, at + 2 * S::kTile);
        at += kWaves * 1024;
        row += kRowsAll;
      }
    }
  };
  issue(W.c0, 0);
  Rows<D> w;
  constexpr int kTiles = 2 * RW / kWaves;  // of 32 keys, of a stage, for a wave
  const uint32_t r0 = W.row0 + 32 * (wave % RW) + l32, first = kTiles == 1 ? wave / RW : 0;
  load_rows_of(w, P, W, r0, h);
  uint32_t buf = 0;
#pragma unroll 1
  for (uint32_t base = W.c0; base < W.c1; base += kStageKeys, buf ^= 1) {
    wait_vmcnt<0>();  // this wave's copies of the stage
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // everyone's; and everyone has read the stage before
    asm volatile("" ::: "memory");
    if (base + kStageKeys < W.c1) issue(base + kStageKeys, buf ^ 1);
    const uint32_t kt = lds0 + buf * 4 * S::kTile + first * S::kTile, vt = kt + 2 * S::kTile;
    const int left = W.c1 - base - 32 * first;
    auto turn = [&](auto second) __attribute__((always_inline)) {
      f32x16 s[kTiles];
#pragma unroll
      for (int n = 0; n < kTiles; n++) scores(w, Keys<D>(kt + n * S::kTile, l32, h), s[n]);
      if (left < 32 * kTiles) {
#pragma unroll
        for (int n = 0; n < kTiles; n++) {
          mask_scores(s[n], left - 32 * n, h);
          clear_values<D>(vt + n * S::kTile, left - 32 * n, lane);  // the waves store the same, each before it reads the rows
        }
      }
      const bool again = settle(w, s, second, [&] {
#pragma unroll
        for (int n = 0; n < kTiles; n++) mend_scores(w, Keys<D>(kt + n * S::kTile, l32, h), s[n]);
      });
      half8 ph[2 * kTiles], pl[2 * kTiles];
      weigh<D, kTiles>(w, s, ph, pl);
      add_values<D, kTiles>(w, vt, ph, pl, lane);
      return again;
    };
    if (__builtin_expect(turn(std::false_type{}), 0)) turn(std::true_type{});
  }
  mend_values(w, W.k, W.v, RS, W.c0, W.c1, first, kTiles == 1 ? 2 : 1, lane);
  w.l = swap_sum(w.l);
  if constexpr (kTiles == 1) {
    join_waves<D, 2>(w, W, lds, wave, lane);
    return;
  }
  if (r0 >= W.n_rows) return;
  float4* const acc = W.acc + wave * 32 * (D / 4);
#pragma unroll
  for (int d = 0; d < S::DT; d++)
#pragma unroll
    for (int i = 0; i < 4; i++)
      acc[((4 * d + i) * 2 + h) * 32 + l32] =
          make_float4(w.acc[d][4 * i], w.acc[d][4 * i + 1], w.acc[d][4 * i + 2], w.acc[d][4 * i + 3]);
  if (h == 0) W.ml[wave * 32 + l32] = make_float2(ldexpf(w.m, -w.e), w.l);
}

// grid: the prefixes' workgroups, then the members' own rows'; KV head fastest
// (with 8 KV heads a head's workgroups run on one XCD and share its L2).  RW: tiles of
// 32 query rows that a prefix's workgroup takes, 1, 2 or 4.
template <int D, int RW>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_partial_kernel(const Params P) {
  extern __shared__ __align__(256) unsigned char lds[];
  Work W;
  uint32_t b = blockIdx.x;
  if (b < P.n_prefix_wgs) {
    W.kvh = b % P.n_kv;
    b /= P.n_kv;
    const uint32_t n_rg = (P.tiles + RW - 1) / RW, rg = b % n_rg;
    b /= n_rg;
    const uint32_t slot = b;
    uint32_t g, c, rows, chunk;
    if (!P.shared) {
      g = slot / P.cp, c = slot % P.cp;
      rows = rows_of(P.prefix_len, g, P.max_prefix);
      chunk = chunk_of(rows, P.cp);
    } else {
      const Shares a = shares_of(P, threadIdx.x & 63);
      g = __builtin_popcountll(__ballot(a.upto <= slot));
      if (g >= P.n_groups) return;
      c = slot - lane_of(a.upto - a.n, g);
      rows = lane_of(a.rows, g);
      chunk = a.chunk;
    }
    W.c0 = c * chunk;
    W.c1 = min(W.c0 + chunk, rows);
    if (W.c0 >= W.c1) return;
    const size_t at = (static_cast<size_t>(g) * P.max_prefix * P.n_kv + W.kvh) * D;
    W.k = reinterpret_cast<const uint8_t*>(P.k_prefix + at);
    W.v = reinterpret_cast<const uint8_t*>(P.v_prefix + at);
    W.member0 = g * P.n_per;
    W.row0 = rg * 32 * RW;
    W.n_rows = P.R;
    W.stored = 32;
    const size_t part = (static_cast<size_t>(slot) * P.n_kv + W.kvh) * P.tiles + rg * RW;
    W.ml = P.ml_p + part * 32;
    W.acc = P.acc_p + part * 32 * (D / 4);
    if constexpr (RW > 1) {
      many_rows<D, RW>(P, W, lds);
      return;
    }
  } else {
    b -= P.n_prefix_wgs;
    W.kvh = b % P.n_kv;
    b /= P.n_kv;
    const uint32_t tile = b % P.own_tiles;
    b /= P.own_tiles;
    const uint32_t c = b % P.co, m = P.sorted ? by_length(P, b / P.co, threadIdx.x & 63) : b / P.co;
    const uint32_t rows = rows_of(P.own_len, m, P.max_own), chunk = chunk_of(rows, P.co);
    W.c0 = c * chunk;
    W.c1 = min(W.c0 + chunk, rows);
    if (W.c0 >= W.c1) return;
    const size_t at = (static_cast<size_t>(m) * P.max_own * P.n_kv + W.kvh) * D;
    W.k = reinterpret_cast<const uint8_t*>(P.k_own + at);
    W.v = reinterpret_cast<const uint8_t*>(P.v_own + at);
    W.member0 = m;
    W.row0 = tile * 32;
    W.n_rows = P.G;
    W.stored = P.own_rows;
    const size_t part = ((static_cast<size_t>(m) * P.co + c) * P.n_kv + W.kvh) * P.own_tiles + tile;
    W.ml = P.ml_o + part * P.own_rows;
    W.acc = P.acc_o + part * P.own_rows * (D / 4);
  }
  few_rows<D>(P, W, lds);
}

// ------------------------------------------------------------------ combine
// out = sum_c acc_c w_c / sum_c l_c w_c, w_c = e^{m_c - m}.  An item is one register
// quad of 32 query rows: lane l has four dims of row l % 32, so a row's maximum and
// sums stay in its lane, and a load of the prefix's results is 1 KB in a row.  W waves
// take an item: wave w chunks w, w + W, .., kBatch loads in flight, then they join in
// fixed order.  Items: KV head fastest, as the partial kernel's workgroups.
template <int D, int W>
__global__ __launch_bounds__(256) void shared_combine_kernel(const Params P, uint32_t n_items) {
  constexpr uint32_t kQuads = D / 8, kBatch = 8;
  __shared__ float4 pa[4][64];
  __shared__ float2 pm[4][64];
  const uint32_t lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % W;
  uint32_t b = blockIdx.x * (4 / W) + wave / W;
  if (b >= n_items) return;  // with W = 4 a workgroup has one item
  const uint32_t kvh = b % P.n_kv;
  b /= P.n_kv;
  const uint32_t quad = b % kQuads;
  b /= kQuads;
  const uint32_t tile = b % P.tiles, g = b / P.tiles;
  const uint32_t r0 = tile * 32 + l32, r = min(r0, P.R - 1);
  const uint32_t m = g * P.n_per + r / P.G, hg = r % P.G;
  float M = -INFINITY, L = 0.f;
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](float2 ml, float4 a) {
    // a part without a reference has no weight, but its NaN stay
    const float ew = ml.x == -INFINITY ? 0.f : factor_of((ml.x - M) * P.scale);
    L = __builtin_fmaf(ml.y, ew, L);
    A.x = __builtin_fmaf(a.x, ew, A.x);
    A.y = __builtin_fmaf(a.y, ew, A.y);
    A.z = __builtin_fmaf(a.z, ew, A.z);
    A.w = __builtin_fmaf(a.w, ew, A.w);
  };
  auto raise = [&](float to) {
    const float keep = M == -INFINITY ? 0.f : factor_of((M - to) * P.scale);
    M = to;
    if (keep != 1.f) L *= keep, A.x *= keep, A.y *= keep, A.z *= keep, A.w *= keep;
  };
  // the first loads are asked for with the lengths: what turns out not to be there is not joined
  const size_t step_p = static_cast<size_t>(P.n_kv) * P.tiles, step_o = static_cast<size_t>(P.n_kv) * P.own_tiles;
  size_t at_p = (static_cast<size_t>(g) * P.cp * P.n_kv + kvh) * P.tiles + tile;
  const size_t at_o = (static_cast<size_t>(m) * P.co * P.n_kv + kvh) * P.own_tiles + hg / 32;
  float2 ml[kBatch], ml_o = make_float2(-INFINITY, 0.f);
  float4 a[kBatch], a_o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto load = [&](uint32_t c, uint32_t last) {
#pragma unroll
    for (uint32_t j = 0; j < kBatch; j++) {
      const size_t o = (at_p + min(c + W * j, last) * step_p) * 32;
      ml[j] = P.ml_p[o + l32];
      a[j] = P.acc_p[o * (D / 4) + (quad * 2 + h) * 32 + l32];
    }
  };
  auto load_own = [&](uint32_t c) {
    const size_t o = (at_o + c * step_o) * P.own_rows;
    ml_o = P.ml_o[o + hg % 32];
    a_o = P.acc_o[o * (D / 4) + (quad * 2 + h) * P.own_rows + hg % 32];
  };
  if (part < P.co) load_own(part);
  if (part < P.cp) load(part, P.cp - 1);  // cp is 0 where the chunks are shared
  const uint32_t plen = P.prefix_len ? P.prefix_len[g] : 0, olen = P.own_len ? P.own_len[m] : 0;
  const bool fits = plen <= P.max_prefix && olen <= P.max_own;
  if (plen && plen <= P.max_prefix) {
    uint32_t n;
    if (!P.shared) {
      const uint32_t chunk = chunk_of(plen, P.cp);
      n = (plen + chunk - 1) / chunk;
    } else {
      const Shares sh = shares_of(P, lane);
      n = lane_of(sh.n, g);
      at_p += lane_of(sh.upto - sh.n, g) * step_p;
    }
    for (uint32_t c = part; c < n; c += W * kBatch) {
      if (c != part || P.shared) load(c, n - 1);
      float mx = M;
#pragma unroll
      for (uint32_t j = 0; j < kBatch; j++)
        if (c + W * j < n) mx = __builtin_elementwise_maximum(mx, ml[j].x);
      raise(mx);
#pragma unroll
      for (uint32_t j = 0; j < kBatch; j++)
        if (c + W * j < n) join(ml[j], a[j]);
    }
  }
  if (olen && olen <= P.max_own) {
    const uint32_t chunk = chunk_of(olen, P.co), n = (olen + chunk - 1) / chunk;
    for (uint32_t c = part; c < n; c += W) {
      if (c != part) load_own(c);
      raise(__builtin_elementwise_maximum(M, ml_o.x));
      join(ml_o, a_o);
    }
  }
  if constexpr (W > 1) {
    pa[wave][lane] = A;
    pm[wave][lane] = make_float2(M, L);
    whd::lds_barrier();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < W; w++) M = __builtin_elementwise_maximum(M, pm[w][lane].x);
    L = 0.f;
    A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; w++) join(pm[w][lane], pa[w][lane]);
  }
  if (r0 >= P.R) return;
  f32x4u v = f32x4u{A.x, A.y, A.z, A.w} / L;  // no key's score above -inf: 0 / 0, as the formula
  if (!fits || (plen | olen) == 0) {
    const float fill = fits ? 0.f : __builtin_nanf("");
    v = f32x4u{fill, fill, fill, fill};
  }
  *reinterpret_cast<f32x4u*>(P.out + (static_cast<size_t>(m) * P.n_heads + kvh * P.G + hg) * D + 32 * (quad >> 2) +
                             8 * (quad & 3) + 4 * h) = v;
}

// ------------------------------------------------------------------ launching
size_t al256(size_t v) { return (v + 255) / 256 * 256; }
size_t div_up(size_t a, size_t b) { return (a + b - 1) / b; }
size_t clamp(size_t v, size_t lo, size_t hi) { return v < lo ? lo : v > hi ? hi : v; }

Params plan(size_t n_groups, size_t n_per, size_t n_heads, size_t n_kv, size_t D, size_t max_prefix, size_t max_own) {
  Params P{};
  P.n_groups = static_cast<uint32_t>(n_groups);
  P.n_per = static_cast<uint32_t>(n_per);
  P.max_prefix = static_cast<uint32_t>(max_prefix);
  P.max_own = static_cast<uint32_t>(max_own);
  P.n_heads = static_cast<uint32_t>(n_heads);
  P.n_kv = static_cast<uint32_t>(n_kv);
  P.G = static_cast<uint32_t>(n_heads / n_kv);
  P.R = static_cast<uint32_t>(n_per) * P.G;
  P.tiles = (P.R + 31) / 32;
  P.own_tiles = (P.G + 31) / 32;
  P.own_rows = P.G < 32 ? P.G : 32;
  P.scale = kLog2e / sqrtf(static_cast<float>(D));
  const size_t members = n_groups * n_per, cus = static_cast<size_t>(wh::cu_count());
  // Prefix.  Work: 128 keys of a tile per CU.  Little work: 32 query rows to a workgroup, one
  // workgroup per CU, as few partial results.  More: 64 or 128 rows to a workgroup, whose
  // stages are read from the L2 once for all of them (where the rows fill it), then two
  // workgroups per CU, so that one's products run beside the other's exponentials, unless the
  // members' own rows, which memory bounds, need the second place.  A call in us, 32 / 8 heads
  // of 128, with 32, 64 and 128 rows at one / at two workgroups per CU:
  //   members  prefix  own  work       32           64          128
  //        32    4000    0     4  17.3 / 18.6  18.0 / 17.8  20.6 / 20.6
  //        64    6000    0    12  31.0 / 29.6  30.4 / 29.5  28.9 / 32.0
  //        64    6000  350    12  42.6 / 47.9  40.8 / 47.7  44.4 / 46.4
  //        48   12000    0    18  37.5 / 35.7  37.5 / 35.4  38.0 / 38.2
  //        64   20000  350    39  85.0 / 82.8  78.9 / 81.8  69.9 / 79.1
  //        48   60000  350    88  152 / 133    140 / 125    151 / 137
  //        64   40000  350    78  145 / 131    134 / 121    123 / 118
  //        16   60000   50    29  63.5 / 65.6  61.0 / 59.1  82.7 / 76.4
  //        48  131000  400   192  323 / 273    293 / 258    319 / 285
  //        40   60000    0    73  129 / 115    134 / 119    145 / 132  (5 tiles)
  // 32 / 4 heads of 64, whose rows are half as long:
  //        16    4000    0     2  10.6 / 11.8  12.0 / 12.2  13.0 / 13.1
  //        32   16000  100    16  24.2 / 21.8  24.1 / 23.8  22.9 / 25.1
  //        24   60000  100    44  53.5 / 43.2  51.9 / 44.7  55.7 / 49.8
  //        32   60000  400    59  64.5 / 54.3  62.2 / 51.1  54.6 / 49.6
  auto work_of = [&](size_t rows_of_32, size_t keys) {
    return static_cast<double>(rows_of_32) * static_cast<double>(keys) / (128.0 * static_cast<double>(cus));
  };
  const double work = work_of(n_groups * n_kv * P.tiles, max_prefix), work_own = work_of(members * n_kv * P.own_tiles, max_own);
  const uint32_t of_four = (P.tiles + 3) / 4 * 4, of_two = (P.tiles + 1) / 2 * 2;
  if (D == 128) P.rw = work < 10.0 ? 1 : 4 * of_four <= 5 * P.tiles && 4.0 * work_own <= work ? 4 : 8 * of_two <= 9 * P.tiles ? 2 : 1;
  else P.rw = 4 * of_four <= 5 * P.tiles && work >= 24.0 ? 4 : 1;
  const double two_from = D == 64 ? P.rw == 4 ? 0.0 : 7.0 : P.rw == 4 ? 56.0 : P.rw == 2 ? 16.0 : 20.0;
  const bool two = (P.rw > 1 || P.tiles >= 3) && work >= two_from && 10.0 * work_own <= work;
  const size_t each = n_kv * ((P.tiles + P.rw - 1) / P.rw), wanted = (two ? 2 : 1) * cus / each;
  const size_t least = P.rw == 1 ? kLeastChunk : 256;
  P.cp = max_prefix == 0 ? 0 : static_cast<uint32_t>(clamp(wanted / n_groups, 1, div_up(max_prefix, least)));
  P.slots = static_cast<uint32_t>(n_groups) * P.cp;
  // Several prompts are seldom of one length.  Chunks planned from the lengths cost each workgroup
  // 1 us of looking at all of them, so they need some work.  In us, cp chunks each / shared, of
  // equal lengths, of any up to the longest, of lengths that fall by a factor:
  //   6 groups x 5 members, 12000, 64 dims    32.1 / 32.6   28.8 / 25.1   24.0 / 15.4
  //   6 x 5, 12000, 128 dims                  67.7 / 68.0   54.2 / 49.1   38.6 / 21.9
  //   16 x 4, 4000, 128 dims                  63.9 / 67.3   46.5 / 45.4   36.2 / 29.4
  //   32 x 1, 6000, 128 dims                  144 / 147     109 / 104     76.2 / 34.3
  //   3 x 4, 1100, 128 dims (work 1)          15.4 / 16.0   13.7 / 14.3   11.5 / 13.8
  //   8 x 8, 4000, 64 dims (work 4)           16.5 / 17.4   15.6 / 16.3   14.7 / 15.7
  const size_t shared = wanted >= 2 * n_groups ? wanted : 2 * wanted;
  if (n_groups > 1 && n_groups <= 64 && shared >= 2 * n_groups && work >= kShareFrom && max_prefix < 1u << 27) {
    P.shared = 1;
    P.cp = 0;
    P.slots = static_cast<uint32_t>(shared);
  }
  P.n_prefix_wgs = static_cast<uint32_t>(each * P.slots);
  const size_t own = members * n_kv * P.own_tiles;
  P.co = max_own == 0 ? 0 : static_cast<uint32_t>(clamp(cus / own, 1, div_up(max_own, kLeastChunk)));
  // More own workgroups than are there at once: the longest first, so that none of them is left at
  // the end.  32 / 8 heads of 128, own rows of any number up to: 48 members at 6000, 500: 34.1 ->
  // 30.9 us, 64 at 6000, 700: 51.4 -> 49.0, 64 at 900, 1500: 62.2 -> 57.0; of one number 45.0 -> 46.9,
  // 64.5 -> 65.7, 83.8 -> 83.9.
  P.sorted = members <= 64 && own * P.co >= cus;
  return P;
}

// Lays the workspace out (offsets only where base is null); returns its size.
size_t layout(Params& P, size_t D, void* base) {
  char* b = static_cast<char*>(base);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* r = b ? b + off : nullptr;
    off += al256(bytes);
    return r;
  };
  const size_t p = static_cast<size_t>(P.slots) * P.n_kv * P.tiles * 32;
  const size_t o = static_cast<size_t>(P.n_groups) * P.n_per * P.co * P.n_kv * P.own_tiles * P.own_rows;
  P.ml_p = reinterpret_cast<float2*>(take(8 * p));
  P.acc_p = reinterpret_cast<float4*>(take(4 * D * p));
  P.ml_o = reinterpret_cast<float2*>(take(8 * o));
  P.acc_o = reinterpret_cast<float4*>(take(4 * D * o));
  return off;
}

template <int D, int RW>
int launch_partial(const Params& P, size_t wgs, hipStream_t s) {
  WH_ENSURE_LDS(static_cast<size_t>(Shape<D>::kLds), &shared_partial_kernel<D, RW>);
  shared_partial_kernel<D, RW><<<static_cast<unsigned>(wgs), 64 * kWaves, Shape<D>::kLds, s>>>(P);
  WH_LAUNCH_CHECK("shared attention kernel launch");
  return WH_OK;
}

template <int D>
int launch_all(const Params& P, hipStream_t s) {
  const size_t own = static_cast<size_t>(P.n_groups) * P.n_per * P.co * P.n_kv * P.own_tiles;
  const size_t wgs = P.n_prefix_wgs + own;
  if (wgs) {
    int st;
    if (P.rw == 1) st = launch_partial<D, 1>(P, wgs, s);
    else if (D == 64 || P.rw == 4) st = launch_partial<D, 4>(P, wgs, s);
    else if constexpr (D == 128) st = launch_partial<D, 2>(P, wgs, s);
    if (st) return st;
  }
  const size_t items = static_cast<size_t>(P.n_groups) * P.n_kv * P.tiles * (D / 8);
  if (items <= 8 * static_cast<size_t>(wh::cu_count()))
    shared_combine_kernel<D, 4><<<static_cast<unsigned>(items), 256, 0, s>>>(P, static_cast<uint32_t>(items));
  else
    shared_combine_kernel<D, 1><<<static_cast<unsigned>((items + 3) / 4), 256, 0, s>>>(P, static_cast<uint32_t>(items));
  WH_LAUNCH_CHECK("shared attention combine launch");
  return WH_OK;
}

}  // namespace

namespace wh {

bool shared_attention_shape_ok(size_t n_groups, size_t n_per, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                               size_t max_prefix, size_t max_own) {
  if ((head_dim != 64 && head_dim != 128) || n_kv_heads == 0 || n_heads == 0 || n_heads > 1024 || n_heads % n_kv_heads != 0 ||
      n_groups > kMaxMembers || n_per > kMaxMembers || n_groups * n_per > kMaxMembers || max_prefix >> 31 || max_own >> 31)
    return false;
  // the join's launch: a wave per item, fewer than 2^32 threads
  const size_t tiles = div_up(n_per * (n_heads / n_kv_heads), 32);
  return !(n_groups * n_kv_heads * tiles * (head_dim / 8) * 64 >> 32);
}

size_t shared_attention_workspace_bytes(size_t n_groups, size_t n_per, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                        size_t max_prefix, size_t max_own) {
  Params P = plan(n_groups, n_per, n_heads, n_kv_heads, head_dim, max_prefix, max_own);
  return layout(P, head_dim, nullptr);
}

int launch_shared_attention(const SharedAttnArgs& a, void* workspace, hipStream_t s) {
  Params P = plan(a.n_groups, a.n_per, a.n_heads, a.n_kv_heads, a.head_dim, a.max_prefix, a.max_own);
  layout(P, a.head_dim, workspace);
  P.q = a.q, P.ldq = a.ldq;
  P.prefix_len = a.max_prefix ? a.prefix_len : nullptr;
  P.own_len = a.max_own ? a.own_len : nullptr;
  P.k_prefix = static_cast<const _Float16*>(a.k_prefix), P.v_prefix = static_cast<const _Float16*>(a.v_prefix);
  P.k_own = static_cast<const _Float16*>(a.k_own), P.v_own = static_cast<const _Float16*>(a.v_own);
  P.out = a.out;
  return a.head_dim == 128 ? launch_all<128>(P, s) : launch_all<64>(P, s);
}

}  // namespace wh

WH_API size_t wh_attention_shared_workspace_bytes(size_t n_groups, size_t n_per, size_t n_heads, size_t n_kv_heads,
                                                  size_t head_dim, size_t max_prefix, size_t max_own) {
  if (n_groups == 0 || n_per == 0 ||
      !wh::shared_attention_shape_ok(n_groups, n_per, n_heads, n_kv_heads, head_dim, max_prefix, max_own))
    return 0;
  return wh::shared_attention_workspace_bytes(n_groups, n_per, n_heads, n_kv_heads, head_dim, max_prefix, max_own);
}

WH_API int wh_attention_shared(const float* q, size_t ldq, const uint32_t* prefix_len, const uint32_t* own_len,
                               size_t n_groups, size_t n_per, const void* k_prefix, const void* v_prefix,
                               size_t max_prefix, const void* k_own, const void* v_own, size_t max_own, size_t n_heads,
                               size_t n_kv_heads, size_t head_dim, float* out, void* workspace, size_t workspace_bytes,
                               wh_stream_t stream) {
  const char* const fn = "attention_shared";
  if (!wh::shared_attention_shape_ok(n_groups, n_per, n_heads, n_kv_heads, head_dim, max_prefix, max_own))
    return wh::set_error(WH_ERR_INVALID_SHAPE,
                         "%s: head_dim %zu, %zu heads, %zu KV heads, %zu x %zu members, %zu and %zu rows not supported", fn,
                         head_dim, n_heads, n_kv_heads, n_groups, n_per, max_prefix, max_own);
  if (ldq < n_heads * head_dim)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: row stride %zu below the rows' %zu elements", fn, ldq, n_heads * head_dim);
  if (n_groups == 0 || n_per == 0) return WH_OK;
  if (!q || !out || (max_prefix && (!prefix_len || !k_prefix || !v_prefix)) || (max_own && (!own_len || !k_own || !v_own)))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  const void* caches[] = {k_prefix, v_prefix, k_own, v_own, workspace};
  for (const void* p : caches)
    if (!wh::aligned(p, 16))
      return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: caches and workspace must be 16-byte aligned", fn);
  const void* ptrs[] = {q, out, prefix_len, own_len};
  for (const void* p : ptrs)
    if (!wh::aligned(p, 4)) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: arrays must be 4-byte aligned", fn);
  const size_t need = wh::shared_attention_workspace_bytes(n_groups, n_per, n_heads, n_kv_heads, head_dim, max_prefix, max_own);
  if (workspace_bytes < need || (need && !workspace))
    return wh::set_error(WH_ERR_BUFFER_TOO_SMALL, "%s: workspace too small: needed %zu bytes, available %zu", fn, need,
                         workspace ? workspace_bytes : static_cast<size_t>(0));
  const wh::SharedAttnArgs a{q,     ldq,   prefix_len, own_len, n_groups,   n_per,    k_prefix, v_prefix, max_prefix,
                             k_own, v_own, max_own,    n_heads, n_kv_heads, head_dim, out};
  return wh::launch_shared_attention(a, workspace, reinterpret_cast<hipStream_t>(stream));
}
