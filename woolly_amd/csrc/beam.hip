// beam.hip -- the choice of a beam search over beams and vocabulary, and what
// belongs to the beams following them, on gfx950.
//
// Selection.  Beam b continued by token i has s = score_b + l_i - lse_b,
// lse_b = log sum_j exp l_j; of a sequence's continuations the n_out with the
// highest s / count^alpha are wanted, in order.  Two launches:
//   1. a workgroup per 8192 logits of a beam: the sum of their exponentials
//      relative to the largest, and the n_out highest logits
//   2. a workgroup per sequence: the beams' lse, the n_out best of all chunks'
//      lists, and the histories
// Ranks are made by counting.  Among the 64 largest logits of a wave's lanes the
// n_out-th is a bound that at least n_out logits reach; the highest of the waves'
// bounds (halved on until it does) leaves a few dozen logits of a chunk, and the
// place of each is the number of those before it.  Logits that are equal come in
// the order of their tokens: the keys that are compared hold both.  Where too many
// are equal for that they are taken one maximum at a time.
// lse in 64 bits: the few highest terms, which make the sum, are exponentials in
// 64 bits, the others in 32 bits summed in 64.
//
// Reordering.  A thread holds one 16-byte column of a state's rows for all beams:
// it loads what its moved beams take before it stores any of it, so rows move in
// place, whatever the parents are.
#include <algorithm>
#include <memory>
#include <new>
#include <type_traits>

#include "members.hpp"
#include "tree.hpp"

namespace {

constexpr uint32_t kNoToken = 0xFFFFFFFFu;
constexpr int kThreads = 512;                 // of the first launch
constexpr int kPer = 16;                      // logits per thread
constexpr int kChunk = kThreads * kPer;
constexpr uint32_t kList = 128;               // logits of a chunk that are ranked, 2 n_out or more
constexpr int kPickThreads = 1024;
constexpr uint32_t kPickList = 1024;

// The order of floats as that of unsigned numbers; nothing for what is not allowed.
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value32(uint32_t o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ unsigned long long order64(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double value64(unsigned long long o) {
  return __builtin_bit_cast(double, o >> 63 ? o & ~(1ull << 63) : ~o);
}

// A bound that at least n of the lanes' numbers reach, 0 where fewer than n lanes have
// one above 0: the n-th largest of them, cut to its upper kBits bits.
template <int kBits>
__device__ __forceinline__ uint32_t nth_largest(uint32_t v, uint32_t n) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 32 - kBits; bit--) {
    const uint32_t with = t | 1u << bit;
    if (static_cast<uint32_t>(__builtin_popcountll(__ballot(v >= with))) >= n) t = with;
  }
  return t;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  return whd::wave_join(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const unsigned long long o = __shfl_xor(v, off, 64);
    v = o > v ? o : v;
  }
  return v;
}
// Sum over the wave's 64 lanes, in every lane: swaps within rows of 16 lanes, then of
// rows and halves (as wave_join, tree.hpp).
__device__ __forceinline__ double wave_sum_f64(double v) {
  auto lo = [](double x) { return static_cast<uint32_t>(__builtin_bit_cast(unsigned long long, x)); };
  auto hi = [](double x) { return static_cast<uint32_t>(__builtin_bit_cast(unsigned long long, x) >> 32); };
  auto make = [](uint32_t l, uint32_t h) { return __builtin_bit_cast(double, static_cast<unsigned long long>(h) << 32 | l); };
  auto dpp = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  auto step = [&](auto ctrl) { v += make(dpp(lo(v), ctrl), dpp(hi(v), ctrl)); };
  step(std::integral_constant<int, 0xB1>{});
  step(std::integral_constant<int, 0x4E>{});
  step(std::integral_constant<int, 0x141>{});
  step(std::integral_constant<int, 0x140>{});
  const auto l16 = __builtin_amdgcn_permlane16_swap(lo(v), lo(v), false, false), h16 = __builtin_amdgcn_permlane16_swap(hi(v), hi(v), false, false);
  v = make(l16[0], h16[0]) + make(l16[1], h16[1]);
  const auto l32 = __builtin_amdgcn_permlane32_swap(lo(v), lo(v), false, false), h32 = __builtin_amdgcn_permlane32_swap(hi(v), hi(v), false, false);
  return make(l32[0], h32[0]) + make(l32[1], h32[1]);
}

struct Params {
  const float* logits;
  size_t ld;
  uint32_t vocab, n_seqs, n_beams, n_out, n_chunks;
  const float* scores;
  const uint32_t* last;    // null: none has ended
  uint32_t end_token;
  float alpha;
  const uint32_t* counts;
  const uint32_t* len;
  float* scores_out;
  uint32_t *tokens, *parents, *counts_out, *history, *len_out;
  size_t history_stride;
  // workspace
  double* sums;            // [rows][n_chunks]: of exp(l - the chunk's largest)
  uint2* lists;            // [rows][n_chunks][n_out]: (order of the logit, token), best first; order 0: none
};

// What a beam is in this step.
enum { kGone, kOpen, kEnded };
__device__ __forceinline__ int state_of(const Params& P, uint32_t row) {
  const float s = P.scores[row];
  if (!(s > -INFINITY && s < INFINITY)) return kGone;
  return P.last && P.last[row] == P.end_token ? kEnded : kOpen;
}

// grid: (n_chunks, rows).  Thread t has logits 4 t .. 4 t + 3 of each 4 kThreads
// (VEC: rows 16-byte aligned) or t, t + kThreads, ..
template <bool VEC>
__global__ __launch_bounds__(kThreads) void beam_chunk_kernel(const Params P) {
  constexpr int kWaves = kThreads / 64;
  __shared__ unsigned long long list[kList];
  __shared__ uint32_t tops[kWaves], bounds[kWaves], counts[kWaves];
  __shared__ unsigned long long red64[kWaves];
  __shared__ double rests[kWaves], terms[kList];
  __shared__ uint32_t n_list;
  const uint32_t row = blockIdx.y, t = threadIdx.x, lane = t & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  if (state_of(P, row) != kOpen) return;
  const uint32_t i0 = blockIdx.x * kChunk, n = min(P.vocab - i0, static_cast<uint32_t>(kChunk));
  auto at = [&](int j) -> uint32_t { return VEC ? 4 * t + (j & 3) + 4 * kThreads * (j >> 2) : t + kThreads * j; };
  const float* p = P.logits + row * P.ld + i0;
  float x[kPer];  // -inf: not allowed, or not there
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < kPer; j += 4) {
      const uint32_t a = at(j);
      if (a + 4 <= n) {
        const float4 v = *reinterpret_cast<const float4*>(p + a);
        x[j] = v.x, x[j + 1] = v.y, x[j + 2] = v.z, x[j + 3] = v.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[j + k] = a + k < n ? p[a + k] : -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; j++) x[j] = at(j) < n ? p[at(j)] : -INFINITY;
  }
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    x[j] = fmaxf(x[j], -INFINITY);  // NaN: -inf
    top = fmaxf(top, x[j]);
  }
  if (t == 0) n_list = 0;
  const uint32_t key = top > -INFINITY ? order32(top) : 0u;
  const uint32_t bound = nth_largest<20>(key, P.n_out), wave_top = wave_max_u32(key);
  if (lane == 0) tops[wave] = wave_top, bounds[wave] = bound;
  __syncthreads();
  uint32_t most = 0, least = order32(-3.402823466e38f);
#pragma unroll
  for (int w = 0; w < kWaves; w++) most = max(most, tops[w]), least = max(least, bounds[w]);
  const size_t chunk = static_cast<size_t>(row) * P.n_chunks + blockIdx.x;
  uint2* const out = P.lists + chunk * P.n_out;
  if (most == 0) {
    if (t == 0) P.sums[chunk] = 0.0;
    if (t < P.n_out) out[t] = make_uint2(0, kNoToken);
    return;
  }
  const float m = value32(most);
  auto key_of = [&](int j) { return static_cast<unsigned long long>(order32(x[j])) << 32 | (0xFFFFFFFFu - (i0 + at(j))); };
  // what reaches the bound into the list
  auto gather = [&](float from) __attribute__((always_inline)) {
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; j++) mine += x[j] >= from;
    if (mine == 0) return;
    uint32_t place = atomicAdd(&n_list, mine);
#pragma unroll
    for (int j = 0; j < kPer; j++)
      if (x[j] >= from) {
        if (place < kList) list[place] = key_of(j);
        place++;
      }
  };
  float from = value32(least);
  gather(from);
  auto rest_below = [&](float to) __attribute__((always_inline)) {
    float rest = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      const float e = __builtin_amdgcn_exp2f((x[j] - m) * 1.4426950408889634f);
      rest += x[j] < to ? e : 0.f;
    }
    const double sum = wave_sum_f64(rest);
    if (lane == 0) rests[wave] = sum;
  };
  rest_below(from);
  __syncthreads();
  uint32_t c = n_list;
  if (__builtin_expect(c > kList, 0)) {
    // the bound halved on: at `least` n_out or more, above `up` fewer (or all the same)
    auto count = [&](float f) __attribute__((always_inline)) {
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < kPer; j++) mine += __builtin_popcountll(__ballot(x[j] >= f));
      __syncthreads();
      if (lane == 0) counts[wave] = mine;
      __syncthreads();
      uint32_t all = 0;
#pragma unroll
      for (int w = 0; w < kWaves; w++) all += counts[w];
      return all;
    };
    for (uint32_t up = most; c > kList && up - least > 1;) {
      const uint32_t mid = least + (up - least) / 2, n_mid = count(value32(mid));
      if (n_mid >= P.n_out) least = mid, c = n_mid; else up = mid;
    }
    from = value32(least);
    __syncthreads();
    if (t == 0) n_list = 0;
    __syncthreads();
    if (c <= kList) gather(from);
    rest_below(c <= kList ? from : INFINITY);
    __syncthreads();
  }
  if (c <= kList) {
    // a thread's place is the number of those before it; the sum is made in their order (the
    // list's own is whichever came first)
    if (t < kList) {
      if (t >= c && t < P.n_out) out[t] = make_uint2(0, kNoToken);
      if (t < c) {
        const unsigned long long k = list[t];
        uint32_t before = 0;
        for (uint32_t j = 0; j < c; j++) before += list[j] > k;
        if (before < P.n_out) out[before] = make_uint2(static_cast<uint32_t>(k >> 32), 0xFFFFFFFFu - static_cast<uint32_t>(k));
        terms[before] = exp(static_cast<double>(value32(static_cast<uint32_t>(k >> 32))) - static_cast<double>(m));
      }
    }
    __syncthreads();
    if (wave == 0) {
      double sum = 0.0;
#pragma unroll
      for (uint32_t i = lane; i < kList; i += 64)
        if (i < c) sum += terms[i];
      sum = wave_sum_f64(sum);
#pragma unroll
      for (int w = 0; w < kWaves; w++) sum += rests[w];
      if (lane == 0) P.sums[chunk] = sum;
    }
    return;
  }
  // too many that are equal: the highest below the last one, n_out times
  if (t == 0) {
    double sum = 0.0;
    for (int w = 0; w < kWaves; w++) sum += rests[w];
    P.sums[chunk] = sum;
  }
  unsigned long long last = ~0ull;
  for (uint32_t i = 0; i < P.n_out; i++) {
    unsigned long long best = 0;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      const unsigned long long k = key_of(j);
      if (x[j] > -INFINITY && k < last && k > best) best = k;
    }
    best = wave_max_u64(best);
    if (lane == 0) red64[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) best = red64[w] > best ? red64[w] : best;
    __syncthreads();
    last = best;
    if (t == 0) out[i] = make_uint2(static_cast<uint32_t>(best >> 32), 0xFFFFFFFFu - static_cast<uint32_t>(best));
  }
}

// A continuation as it is compared: the order of its rank, then the lowest beam,
// then the beam's own order (the logit's, then the lowest token).
struct Cand {
  unsigned long long rank;
  uint32_t beam, logit, token;
};
__device__ __forceinline__ bool before(Cand a, Cand b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  if (a.beam != b.beam) return a.beam < b.beam;
  if (a.logit != b.logit) return a.logit > b.logit;
  return a.token < b.token;
}

__device__ __forceinline__ unsigned long long rank_of(double s, double norm, float alpha) {
  return order64(alpha == 0.f ? s : s / norm);
}

// grid: n_seqs.  A thread has one of the sequence's lists, or several.
__global__ __launch_bounds__(kPickThreads) void beam_pick_kernel(const Params P) {
  constexpr uint32_t kHead = 4;  // entries of a list that are asked for at once
  __shared__ double lse[wh::kMaxBeams], score[wh::kMaxBeams], norm[wh::kMaxBeams];
  __shared__ int state[wh::kMaxBeams];
  __shared__ uint32_t tops[wh::kMaxBeams];
  __shared__ uint32_t red[kPickThreads / 64];
  __shared__ Cand best[kPickThreads / 64];
  __shared__ Cand list[kPickList];
  __shared__ Cand chosen[2 * wh::kMaxBeams];
  __shared__ uint32_t from[wh::kMaxBeams], have[wh::kMaxBeams];
  __shared__ uint32_t n_list;
  const uint32_t s = blockIdx.x, t = threadIdx.x, lane = t & 63, row0 = s * P.n_beams;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t n_lists = P.n_beams * P.n_chunks, total = n_lists * P.n_out;
  const uint2* const lists = P.lists + static_cast<size_t>(row0) * P.n_chunks * P.n_out;
  const double* const sums = P.sums + static_cast<size_t>(row0) * P.n_chunks;
  // asked for before it is known which of it counts (a beam that has ended wrote none)
  uint2 head[kHead];
  double sum0 = 0.0;
  if (t < n_lists) {
    sum0 = sums[t];
#pragma unroll
    for (uint32_t j = 0; j < kHead; j++) head[j] = j < P.n_out ? lists[static_cast<size_t>(t) * P.n_out + j] : make_uint2(0, kNoToken);
  }
  if (t == 0) n_list = 0;
  if (t < 2 * wh::kMaxBeams) chosen[t] = Cand{0, 0, 0, kNoToken};
  if (t < P.n_beams) {
    const uint32_t row = row0 + t;
    const int st = state_of(P, row);
    const uint32_t count = (P.counts ? P.counts[row] : 0u) + (st == kOpen);
    tops[t] = 0;
    state[t] = st;
    score[t] = P.scores[row];
    norm[t] = P.alpha == 0.f ? 1.0 : pow(static_cast<double>(max(count, 1u)), static_cast<double>(P.alpha));
  }
  __syncthreads();
  // the beams' largest logits, then lse = log of the sum of the chunks' sums
  for (uint32_t i = t; i < n_lists; i += kPickThreads) {
    const uint32_t b = i / P.n_chunks;
    if (state[b] == kOpen) atomicMax(&tops[b], i == t ? head[0].x : lists[static_cast<size_t>(i) * P.n_out].x);
  }
  __syncthreads();
  double* const terms = reinterpret_cast<double*>(list);  // [kPickThreads], a list's part of its beam's sum
  for (uint32_t i0 = 0; i0 < n_lists; i0 += kPickThreads) {
    const uint32_t i = i0 + t, b = i < n_lists ? i / P.n_chunks : 0;
    double term = 0.0;
    if (i < n_lists && state[b] == kOpen) {
      const uint32_t x = i0 == 0 ? head[0].x : lists[static_cast<size_t>(i) * P.n_out].x;
      if (x) term = (i0 == 0 ? sum0 : sums[i]) * exp(static_cast<double>(value32(x)) - static_cast<double>(value32(tops[b])));
    }
    terms[t] = term;
    __syncthreads();
    for (uint32_t b2 = wave; b2 < P.n_beams; b2 += kPickThreads / 64) {  // in fixed order
      const uint32_t lo = max(b2 * P.n_chunks, i0), hi = min((b2 + 1) * P.n_chunks, min(i0 + kPickThreads, n_lists));
      if (lo >= hi) continue;
      double part = 0.0;
      for (uint32_t e = lo + lane; e < hi; e += 64) part += terms[e - i0];
      part = wave_sum_f64(part);
      if (lane == 0) lse[b2] = lo == b2 * P.n_chunks ? part : lse[b2] + part;
    }
    __syncthreads();
  }
  if (t < P.n_beams && state[t] == kOpen) {
    const double l = static_cast<double>(value32(tops[t])) + log(lse[t]);
    if (tops[t] == 0 || !(l < INFINITY)) state[t] = kGone;  // no token is allowed, or one at +inf
    lse[t] = l;
  }
  __syncthreads();
  // entry j of the sequence's list i
  auto cand = [&](uint32_t i, uint32_t j, auto load) {
    const uint32_t b = i / P.n_chunks;
    if (state[b] == kEnded)  // itself, once
      return i % P.n_chunks + j == 0 ? Cand{rank_of(score[b], norm[b], P.alpha), b, 0, P.end_token} : Cand{0, 0, 0, kNoToken};
    if (state[b] == kGone) return Cand{0, 0, 0, kNoToken};
    const uint2 x = load();
    if (x.x == 0) return Cand{0, 0, 0, kNoToken};
    return Cand{rank_of(score[b] + (static_cast<double>(value32(x.x)) - lse[b]), norm[b], P.alpha), b, x.x, x.y};
  };
  auto entry = [&](uint32_t i, uint32_t j) { return cand(i, j, [&] { return lists[static_cast<size_t>(i) * P.n_out + j]; }); };
  // the lists' first entries give a bound that n_out of them reach (on ranks rounded to 32
  // bits); what reaches it stands at the front of its list
  auto coarse = [](const Cand& k) { return k.rank ? order32(static_cast<float>(value64(k.rank))) : 0u; };
  uint32_t top = 0;
  for (uint32_t i = t; i < n_lists; i += kPickThreads) top = max(top, coarse(i == t ? cand(i, 0, [&] { return head[0]; }) : entry(i, 0)));
  const uint32_t bound = nth_largest<24>(top, P.n_out);
  if (lane == 0) red[wave] = bound;
  __syncthreads();
  uint32_t least = 1;
#pragma unroll
  for (int w = 0; w < kPickThreads / 64; w++) least = max(least, red[w]);
  for (uint32_t i = t; i < n_lists; i += kPickThreads) {
    auto put = [&](const Cand& k) {
      if (coarse(k) < least) return false;
      const uint32_t place = atomicAdd(&n_list, 1u);
      if (place < kPickList) list[place] = k;
      return true;
    };
    bool on = true;
    uint32_t j = 0;
    if (i == t) {
#pragma unroll
      for (j = 0; j < kHead; j++) on = on && j < P.n_out && put(cand(i, j, [&] { return head[j]; }));
    }
    for (; on && j < P.n_out; j++) on = put(entry(i, j));
  }
  __syncthreads();
  const uint32_t c = n_list;
  if (c <= kPickList) {
    for (uint32_t i = t; i < c; i += kPickThreads) {
      const Cand k = list[i];
      uint32_t place = 0;
      for (uint32_t j = 0; j < c; j++) place += before(list[j], k);
      if (place < P.n_out) chosen[place] = k;
    }
  } else {  // the first one behind the last, n_out times
    Cand last{~0ull, 0, 0, 0};
    for (uint32_t i = 0; i < P.n_out; i++) {
      Cand mine{0, 0, 0, kNoToken};
      for (uint32_t e = t; e < total; e += kPickThreads) {
        const Cand k = entry(e / P.n_out, e % P.n_out);
        if (k.rank && before(last, k) && (mine.rank == 0 || before(k, mine))) mine = k;
      }
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) {
        const Cand o{__shfl_xor(mine.rank, off, 64), __shfl_xor(mine.beam, off, 64), __shfl_xor(mine.logit, off, 64),
                     __shfl_xor(mine.token, off, 64)};
        if (o.rank && (mine.rank == 0 || before(o, mine))) mine = o;
      }
      if (lane == 0) best[wave] = mine;
      __syncthreads();
      for (int w = 0; w < kPickThreads / 64; w++) {
        const Cand o = best[w];
        if (o.rank && (mine.rank == 0 || before(o, mine))) mine = o;
      }
      __syncthreads();
      if (t == 0) chosen[i] = mine;
      last = mine;
      if (mine.rank == 0) break;
    }
  }
  __syncthreads();
  // what an output may overwrite is read before any of them is written
  const uint32_t o = s * P.n_out + t;
  uint32_t parent = 0, count = 0, len = 0;
  if (t < P.n_out) {
    const Cand k = chosen[t];
    parent = k.rank ? k.beam : min(t, P.n_beams - 1);
    if (k.rank) count = (P.counts ? P.counts[row0 + parent] : 0u) + (state[parent] == kOpen);
    if (P.len) len = P.len[row0 + parent];
    if (t < wh::kMaxBeams) from[t] = parent, have[t] = len;
  }
  __syncthreads();
  if (t < P.n_out) {
    const Cand k = chosen[t];
    float v = -INFINITY;
    if (k.rank) v = static_cast<float>(state[parent] == kEnded ? score[parent] : score[parent] + (static_cast<double>(value32(k.logit)) - lse[parent]));
    P.scores_out[o] = v;
    P.tokens[o] = k.token;
    P.parents[o] = parent;
    if (P.counts_out) P.counts_out[o] = count;
    if (P.len_out) P.len_out[o] = len + 1;
  }
  if (!P.history) return;
  // some columns of the histories at a time: what the beams take of them is read before any is written
  uint32_t most = 0;
  for (uint32_t i = 0; i < P.n_beams; i++) most = max(most, have[i]);
  const size_t end = min(static_cast<size_t>(most) + 1, P.history_stride);
  uint32_t* const h = P.history + static_cast<size_t>(row0) * P.history_stride;
  uint32_t* const tile = reinterpret_cast<uint32_t*>(list);
  const uint32_t columns = sizeof(list) / 4 / P.n_beams;
  for (size_t p0 = 0; p0 < end; p0 += columns) {
    const uint32_t n = static_cast<uint32_t>(min(end - p0, static_cast<size_t>(columns)));
    for (uint32_t e = t; e < n * P.n_beams; e += kPickThreads) {
      const uint32_t i = e / n;
      const size_t p = p0 + e % n;
      uint32_t v = chosen[i].token;
      asm("" : "+v"(v));  // not one load from either place
      if (p < have[i]) v = h[from[i] * P.history_stride + p];
      tile[e] = v;
    }
    __syncthreads();
    for (uint32_t e = t; e < n * P.n_beams; e += kPickThreads) {
      const uint32_t i = e / n;
      const size_t p = p0 + e % n;
      if (p <= have[i] && (p == have[i] || from[i] != i)) h[i * P.history_stride + p] = tile[e];
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------- reorder
// States of one launch: their pointers are kernel arguments.
constexpr int kStates = 128;
struct ReorderParams {
  void* state[kStates];
  const uint32_t *parents, *len;
  size_t pending, max_rows, row_pieces;  // pieces of P bytes
  uint32_t n_beams;
};

// grid: (workgroups over a beam's pieces, states, n_seqs).  NB: room for beams.
template <typename Piece, int NB>
__global__ __launch_bounds__(256) void beam_reorder_kernel(const ReorderParams P) {
  const uint32_t s = blockIdx.z;
  const uint32_t* parents = P.parents + static_cast<size_t>(s) * P.n_beams;
  const uint32_t* len = P.len + static_cast<size_t>(s) * P.n_beams;
  const size_t beam = P.max_rows * P.row_pieces;
  Piece* const base = static_cast<Piece*>(P.state[blockIdx.y]) + s * P.n_beams * beam;
  __shared__ size_t from[NB], n[NB];  // a beam's pieces that move, 0 for one that stays
  if (threadIdx.x < NB) {
    const uint32_t i = threadIdx.x, parent = i < P.n_beams ? parents[i] : i;
    const size_t rows = i < P.n_beams && len[i] > P.pending ? len[i] - P.pending : 0;
    n[i] = parent < P.n_beams && parent != i && rows <= P.max_rows ? rows * P.row_pieces : 0;
    from[i] = n[i] ? parent * beam : 0;
  }
  __syncthreads();
  size_t most = 0;
#pragma unroll
  for (int i = 0; i < NB; i++) most = n[i] > most ? n[i] : most;
  for (size_t c = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; c < most; c += static_cast<size_t>(gridDim.x) * 256) {
    Piece v[NB];
#pragma unroll
    for (int i = 0; i < NB; i++)
      if (c < n[i]) v[i] = base[from[i] + c];
#pragma unroll
    for (int i = 0; i < NB; i++)
      if (c < n[i]) base[i * beam + c] = v[i];
  }
}

size_t chunks_of(size_t vocab) { return (vocab + kChunk - 1) / kChunk; }
size_t al256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

WH_API size_t wh_beam_select_workspace_bytes(const wh_beam_rules* rules, size_t n_seqs, size_t vocab) {
  if (!rules || rules->n_beams == 0 || rules->n_beams > wh::kMaxBeams || rules->n_out > 2 * wh::kMaxBeams || n_seqs == 0 ||
      n_seqs * rules->n_beams > 65535 || n_seqs > 65535 || vocab == 0 || vocab >> 31)
    return 0;
  const size_t out = rules->n_out ? rules->n_out : rules->n_beams, chunks = n_seqs * rules->n_beams * chunks_of(vocab);
  return al256(chunks * sizeof(double)) + chunks * out * sizeof(uint2);
}

WH_API int wh_beam_select(const wh_beam_rules* rules, const float* logits, size_t ld, size_t n_seqs, size_t vocab,
                          const float* scores, float* scores_out, uint32_t* tokens, uint32_t* parents, void* workspace,
                          size_t workspace_bytes, wh_stream_t stream) {
  const char* const fn = "beam_select";
  if (!rules) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null rules", fn);
  const wh_beam_rules& r = *rules;
  const size_t n_out = r.n_out ? r.n_out : r.n_beams;
  if (r.n_beams == 0 || r.n_beams > wh::kMaxBeams || n_out > 2 * wh::kMaxBeams)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: %zu beams (1 to %zu), %zu to choose (at most %zu)", fn, r.n_beams,
                         wh::kMaxBeams, n_out, 2 * wh::kMaxBeams);
  if (n_seqs > 65535 || n_seqs * r.n_beams > 65535 || vocab == 0 || vocab >> 31 || ld < vocab)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: %zu x %zu rows (at most 65535) of %zu logits, %zu apart", fn, n_seqs,
                         r.n_beams, vocab, ld);
  if (!(r.length_penalty - r.length_penalty == 0.f))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: the length penalty must be finite", fn);
  if ((r.history || r.len_out) && (n_out != r.n_beams || !r.len))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: history and len_out need len, and as many chosen as there are beams", fn);
  if (n_seqs == 0) return WH_OK;
  if (!logits || !scores || !scores_out || !tokens || !parents)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  const void* ptrs[] = {logits, scores, scores_out, tokens, parents, r.last_tokens, r.counts, r.counts_out, r.history, r.len, r.len_out};
  for (const void* p : ptrs)
    if (!wh::aligned(p, 4)) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: arrays must be 4-byte aligned", fn);
  if (n_out != r.n_beams && (scores_out == scores || tokens == r.last_tokens || (r.counts_out && r.counts_out == r.counts)))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: an output is its input only with as many chosen as there are beams", fn);
  const size_t need = wh_beam_select_workspace_bytes(rules, n_seqs, vocab);
  if (workspace_bytes < need || !workspace)
    return wh::set_error(WH_ERR_BUFFER_TOO_SMALL, "%s: workspace too small: needed %zu bytes, available %zu", fn, need,
                         workspace ? workspace_bytes : static_cast<size_t>(0));
  if (!wh::aligned(workspace, 16)) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", fn);
  Params P{};
  P.logits = logits, P.ld = ld;
  P.vocab = static_cast<uint32_t>(vocab);
  P.n_seqs = static_cast<uint32_t>(n_seqs), P.n_beams = static_cast<uint32_t>(r.n_beams), P.n_out = static_cast<uint32_t>(n_out);
  P.n_chunks = static_cast<uint32_t>(chunks_of(vocab));
  P.scores = scores;
  P.last = r.last_tokens, P.end_token = r.end_token;
  P.alpha = r.length_penalty;
  P.counts = r.counts, P.len = r.len;
  P.scores_out = scores_out, P.tokens = tokens, P.parents = parents;
  P.counts_out = r.counts_out, P.len_out = r.len_out;
  P.history = r.history, P.history_stride = r.history_stride;
  const size_t rows = n_seqs * r.n_beams;
  P.sums = static_cast<double*>(workspace);
  P.lists = reinterpret_cast<uint2*>(static_cast<char*>(workspace) + al256(rows * P.n_chunks * sizeof(double)));
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(P.n_chunks, static_cast<unsigned>(rows));
  if (wh::aligned(logits, 16) && ld % 4 == 0) beam_chunk_kernel<true><<<grid, kThreads, 0, s>>>(P);
  else beam_chunk_kernel<false><<<grid, kThreads, 0, s>>>(P);
  WH_LAUNCH_CHECK("beam selection launch");
  beam_pick_kernel<<<static_cast<unsigned>(n_seqs), kPickThreads, 0, s>>>(P);
  WH_LAUNCH_CHECK("beam choice launch");
  return WH_OK;
}

namespace {

template <typename Piece>
int launch_reorder(const ReorderParams& P, dim3 grid, hipStream_t s) {
  if (P.n_beams <= 4) beam_reorder_kernel<Piece, 4><<<grid, 256, 0, s>>>(P);
  else if (P.n_beams <= 8) beam_reorder_kernel<Piece, 8><<<grid, 256, 0, s>>>(P);
  else if (P.n_beams <= 16) beam_reorder_kernel<Piece, 16><<<grid, 256, 0, s>>>(P);
  else beam_reorder_kernel<Piece, 32><<<grid, 256, 0, s>>>(P);
  WH_LAUNCH_CHECK("beam reordering launch");
  return WH_OK;
}

}  // namespace

WH_API int wh_beam_reorder(void* const* states, size_t n_states, size_t n_seqs, size_t n_beams, size_t max_rows,
                           size_t row_bytes, const uint32_t* parents, const uint32_t* len, size_t pending,
                           wh_stream_t stream) {
  const char* const fn = "beam_reorder";
  if (row_bytes == 0 || row_bytes % 4 != 0 || row_bytes >> 28)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: rows of %zu bytes must be whole 4-byte pieces, below 2^28 bytes", fn, row_bytes);
  if (n_beams > wh::kMaxBeams || n_seqs > 65535 || max_rows == 0 || max_rows >> 31)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: %zu beams (at most %zu) of %zu sequences (at most 65535), max_rows %zu", fn,
                         n_beams, wh::kMaxBeams, n_seqs, max_rows);
  if (n_states == 0 || n_seqs == 0 || n_beams == 0) return WH_OK;
  if (!states || !parents || !len) return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!wh::aligned(parents, 4) || !wh::aligned(len, 4))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: arrays must be 4-byte aligned", fn);
  const size_t piece = row_bytes % 16 == 0 ? 16 : 4;
  for (size_t i = 0; i < n_states; i++)
    if (!states[i] || !wh::aligned(states[i], piece))
      return wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: state %zu must be non-null and %zu-byte aligned", fn, i, piece);
  size_t bytes;
  if (__builtin_mul_overflow(n_seqs * n_beams * max_rows, row_bytes, &bytes))
    return wh::set_error(WH_ERR_INVALID_SHAPE, "%s: %zu x %zu x %zu rows of %zu bytes are no state", fn, n_seqs, n_beams, max_rows,
                         row_bytes);
  // rows of a state named twice, or shared by two, would be moved twice at once: in order of
  // their addresses every state ends before the next begins
  uintptr_t few[2 * kStates];
  std::unique_ptr<uintptr_t[]> many;
  if (n_states > 2 * kStates) {
    many.reset(new (std::nothrow) uintptr_t[n_states]);
    if (!many) return wh::set_error(WH_ERR_OOM, "%s: no memory for %zu states", fn, n_states);
  }
  uintptr_t* at = many ? many.get() : few;
  for (size_t i = 0; i < n_states; i++) at[i] = reinterpret_cast<uintptr_t>(states[i]);
  std::sort(at, at + n_states);
  for (size_t i = 0; i + 1 < n_states; i++)
    if (at[i + 1] - at[i] < bytes) {
      size_t which = n_states - 1;
      while (reinterpret_cast<uintptr_t>(states[which]) != at[i + 1]) which--;
      return at[i + 1] == at[i]
                 ? wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: state %zu is named twice", fn, which)
                 : wh::set_error(WH_ERR_INVALID_ARGUMENT, "%s: state %zu begins within another (of %zu bytes)", fn, which, bytes);
    }
  if (n_beams == 1) return WH_OK;  // no parent but itself
  ReorderParams P{};
  P.parents = parents, P.len = len;
  P.pending = pending, P.max_rows = max_rows;
  P.row_pieces = row_bytes / piece;
  P.n_beams = static_cast<uint32_t>(n_beams);
  const size_t pieces = max_rows * P.row_pieces;
  for (size_t i0 = 0; i0 < n_states; i0 += kStates) {
    const size_t n = n_states - i0 < kStates ? n_states - i0 : kStates;
    for (size_t i = 0; i < n; i++) P.state[i] = states[i0 + i];
    // the lengths are on the device: workgroups that fill the chip stride over the pieces
    const size_t most = 16 * static_cast<size_t>(wh::cu_count()), wanted = (pieces + 255) / 256;
    const size_t x = most / (n * n_seqs) < 1 ? 1 : most / (n * n_seqs);
    const dim3 grid(static_cast<unsigned>(x < wanted ? x : wanted), static_cast<unsigned>(n), static_cast<unsigned>(n_seqs));
    typedef uint32_t piece16 __attribute__((ext_vector_type(4)));
    const int st = piece == 16 ? launch_reorder<piece16>(P, grid, reinterpret_cast<hipStream_t>(stream))
                               : launch_reorder<uint32_t>(P, grid, reinterpret_cast<hipStream_t>(stream));
    if (st) return st;
  }
  return WH_OK;
}
