// beam.hip -- the choice of a beam search over beams and vocabulary, and what
// belongs to the beams following them, on gfx950.
//
// Selection.  Beam b continued by token i has s = score_b + l_i - lse_b,
// lse_b = log sum_j exp l_j; of a sequence's continuations the n_out with the
// highest s / count^alpha are wanted, in order.  Two launches:
//   1. a workgroup per 4096 logits of a beam: the sum of their exponentials
//      relative to the largest, and the n_out highest logits
//   2. a workgroup per sequence: the beams' lse, the n_out best of all chunks'
//      lists, and the histories
// Ranks are made by counting.  Among the 64 largest logits of a wave's lanes the
// n_out-th is a bound that at least n_out logits reach; the highest of the waves'
// bounds (halved on until it does) leaves a few dozen logits of a chunk, and the
// place of each is the number of those before it.  Logits that are equal come in
// the order of their tokens: the keys that are compared hold both.  Where too many
// are equal for that they are taken one maximum at a time.
// lse: the few highest terms, which make the sum where it is uneven, are exponentials in
// 64 bits, the others f32's (a 64-bit one is a few dozen instructions), 8 to a thread's f32
// sum, the threads' sums in 64.  A distance d to the top is off by 2^-24 d, its product with
// log2 e by as much: lse is off by 3e-8 for usual logits, less than half the last place of an
// f32 score above 1.
// The first launch asks for its 4096 logits once and ranks them with nothing in flight (16 x 8
// beams of 128256 logits, of which 51.2 MB are read and those of ended beams are not, in 17
// us, 3.0 TB/s; 4 of 32000 in 5), the second is bound by its steps that wait for each other,
// however few beams there are (8 beams 7.5 us, 4 beams 5.5: 3 until the bound is there,
// 2 for the ranks and outputs, 1 for the histories).
//
// Reordering.  A thread holds one 16-byte column of a state's rows for all beams:
// it loads what its moved beams take before it stores any of it, so rows move in
// place, whatever the parents are.  Bound by memory: a row is written for each beam that
// moves, and read once for those that share a parent (4 of 8 beams x 500 rows of 2 KB x 64
// states: 262 MB written, 137 MB read past the Infinity Cache, 75 to 79 us, 5.1 TB/s; as calls
// 90; 2 of 4 x 60 rows 5.3 us).
#include <algorithm>
#include <memory>
#include <new>

#include "members.hpp"
#include "tree.hpp"

namespace {

constexpr uint32_t kNoToken = 0xFFFFFFFFu;
constexpr int kThreads = 256;                 // of the first launch
constexpr int kPer = 16;                      // logits per thread
constexpr int kChunk = kThreads * kPer;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kList = 128;               // logits of a chunk that are ranked, 2 n_out or more
constexpr size_t kPickWaves = 16;             // of the second launch, at most
constexpr uint32_t kPickList = 1024;          // continuations that are ranked at once
constexpr uint32_t kPickFew = 160;            // more than so many are worth a closer bound

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
// A bound that at least n of the lanes' numbers reach, N of them to a lane and `most` the
// largest; 0 where fewer than n are above 0.  The n-th largest lies somewhere below `most`:
// the power of two of that distance is found by halving (5 counts), then two more of its
// bits, so that some more than n may reach the bound.
template <int N>
__device__ __forceinline__ uint32_t near_top(const uint32_t (&v)[N], uint32_t most, uint32_t n) {
  auto count = [&](uint32_t from) __attribute__((always_inline)) {
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < N; j++) c += __builtin_popcountll(__ballot(v[j] >= from));
    return c;
  };
  auto below = [&](uint32_t by) __attribute__((always_inline)) { return most > by ? most - by : 1u; };
  if (count(1) < n) return 0;
  int bits = 0;  // a distance of 2^bits - 1 is enough, one bit less is not
#pragma unroll
  for (int step = 16; step >= 1; step >>= 1)
    if (count(below((1u << (bits + step - 1)) - 1u)) < n) bits += step;
  uint32_t by = bits < 31 ? (1u << bits) - 1u : 0xFFFFFFFFu;  // of 31 bits none was counted: all
#pragma unroll
  for (int b = 2; b <= 3; b++)
    if (bits >= b && count(below(by - (1u << (bits - b)))) >= n) by -= 1u << (bits - b);
  return below(by);
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
  float x[kPer], top;  // -inf: not allowed, or not there
  auto load = [&]() __attribute__((always_inline)) {
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
    top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      x[j] = fmaxf(x[j], -INFINITY);  // NaN: -inf
      top = fmaxf(top, x[j]);
    }
  };
  load();
  if (t == 0) n_list = 0;
  if (t < kList) list[t] = 0;
  const uint32_t key = top > -INFINITY ? order32(top) : 0u;
  const uint32_t wave_top = wave_max_u32(key), keys[1] = {key}, bound = near_top(keys, wave_top, P.n_out);
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
  // what reaches the bound goes into the list, and out of x
  auto gather = [&](float from) __attribute__((always_inline)) {
    if (!(top >= from)) return;
#pragma unroll
    for (int j = 0; j < kPer; j++)
      if (x[j] >= from) {
        const uint32_t place = atomicAdd(&n_list, 1u);
        if (place < kList) list[place] = key_of(j);
        x[j] = -INFINITY;
      }
  };
  auto add_rest = [&]() __attribute__((always_inline)) {
    float rest[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kPer; j++) rest[j & 1] += __builtin_amdgcn_exp2f((x[j] - m) * kLog2e);
    const double sum = whd::lanes_sum_f64<64>(rest[0] + rest[1]);
    if (lane == 0) rests[wave] = sum;
  };
  gather(value32(least));
  add_rest();
  __syncthreads();
  uint32_t c = n_list;
  if (__builtin_expect(c > kList, 0)) {
    // the bound halved on: at `least` n_out or more, above `up` fewer (or all the same)
    load();
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
    __syncthreads();
    if (t == 0) n_list = 0;
    if (t < kList) list[t] = 0;
    __syncthreads();
    if (c <= kList) gather(value32(least));
    add_rest();
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
        for (uint32_t j = 0; j < c; j += 8)
#pragma unroll
          for (uint32_t u = 0; u < 8; u++) before += list[j + u] > k;  // 0 behind the last
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
      sum = whd::lanes_sum_f64<64>(sum);
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

// grid: n_seqs, a wave per beam (or several), a lane per chunk's list (or several).
__global__ __launch_bounds__(64 * kPickWaves) void beam_pick_kernel(const Params P) {
  constexpr uint32_t kHead = 4;  // entries of a list that are asked for at once
  __shared__ double lse[wh::kMaxBeams], score[wh::kMaxBeams], per_token[wh::kMaxBeams];
  __shared__ int state[wh::kMaxBeams];
  __shared__ uint32_t count_in[wh::kMaxBeams], len_in[wh::kMaxBeams];
  __shared__ uint32_t red[kPickWaves];
  __shared__ Cand best[kPickWaves];
  __shared__ unsigned long long ranks[kPickList + 8];
  __shared__ uint3 rest[kPickList];  // beam, logit, token
  __shared__ Cand chosen[2 * wh::kMaxBeams];
  __shared__ uint32_t from[wh::kMaxBeams], have[wh::kMaxBeams];
  __shared__ uint32_t n_list;
  const uint32_t s = blockIdx.x, t = threadIdx.x, lane = t & 63, row0 = s * P.n_beams, threads = blockDim.x;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6), n_waves = threads / 64;
  const uint32_t per_beam = P.n_chunks * P.n_out;
  const uint2* const lists = P.lists + static_cast<size_t>(row0) * per_beam;
  auto load_heads = [&](uint32_t b, uint2 (&head)[kHead]) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = 0; j < kHead; j++)
      head[j] = lane < P.n_chunks && j < P.n_out ? lists[static_cast<size_t>(b) * per_beam + lane * P.n_out + j] : make_uint2(0, kNoToken);
  };
  // what an entry of a list is compared by
  auto rank_of = [&](uint32_t b, uint32_t x) __attribute__((always_inline)) {
    const double v = state[b] == kEnded ? score[b] : score[b] + (static_cast<double>(value32(x)) - lse[b]);
    return v * per_token[b];
  };
  if (t == 0) n_list = 0;
  if (t < 2 * wh::kMaxBeams) chosen[t] = Cand{0, 0, 0, kNoToken};
  for (uint32_t i = t; i < kPickList + 8; i += threads) ranks[i] = 0;
  // Every beam's lse, and a bound that n_out of its continuations reach: the n_out-th of its
  // lists' first few.
  uint2 mine[kHead];
  uint32_t my_first[kHead] = {0, 0, 0, 0}, least = 1;
  double my_value[kHead];
  for (uint32_t b = wave; b < P.n_beams; b += n_waves) {
    const uint32_t row = row0 + b;
    const double* const sums = P.sums + static_cast<size_t>(row) * P.n_chunks;
    // asked for before it is known whether it counts (a beam that has ended wrote nothing)
    uint2 head[kHead];
    load_heads(b, head);
    double sum = lane < P.n_chunks ? sums[lane] : 0.0;
    int st = state_of(P, row);
    const float sc = P.scores[row];
    const uint32_t count = P.counts ? P.counts[row] : 0u, len = P.len ? P.len[row] : 0u;
    double l = 0.0;
    if (st == kOpen) {
      uint32_t most = head[0].x;
      for (uint32_t c = lane + 64; c < P.n_chunks; c += 64) most = max(most, lists[static_cast<size_t>(b) * per_beam + c * P.n_out].x);
      most = wave_max_u32(most);
      const double m = value32(most);
      sum = head[0].x ? sum * exp(static_cast<double>(value32(head[0].x)) - m) : 0.0;
      for (uint32_t c = lane + 64; c < P.n_chunks; c += 64) {
        const uint32_t x = lists[static_cast<size_t>(b) * per_beam + c * P.n_out].x;
        if (x) sum += sums[c] * exp(static_cast<double>(value32(x)) - m);
      }
      l = m + log(whd::lanes_sum_f64<64>(sum));
      if (most == 0 || !(l < INFINITY)) st = kGone;  // no token is allowed, or one at +inf
    }
    if (st != kOpen) {
#pragma unroll
      for (uint32_t j = 0; j < kHead; j++) head[j] = make_uint2(0, kNoToken);
      if (st == kEnded && lane == 0) head[0] = make_uint2(1, P.end_token);  // itself, once
    }
    if (lane == 0) {
      const uint32_t tokens = max(count + (st == kOpen), 1u);
      per_token[b] = P.alpha == 0.f ? 1.0 : exp(-static_cast<double>(P.alpha) * log(static_cast<double>(tokens)));
      lse[b] = l;
      score[b] = sc;
      count_in[b] = count;
      len_in[b] = len;
      state[b] = st;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the beam's numbers, for the other lanes
    uint32_t first[kHead];
    double value[kHead];
#pragma unroll
    for (uint32_t j = 0; j < kHead; j++) {
      value[j] = rank_of(b, head[j].x);
      first[j] = head[j].x ? order32(static_cast<float>(value[j])) : 0u;
    }
    least = max(least, near_top(first, wave_max_u32(first[0]), P.n_out));
    if (b == wave) {
#pragma unroll
      for (uint32_t j = 0; j < kHead; j++) mine[j] = head[j], my_first[j] = first[j], my_value[j] = value[j];
    }
  }
  if (lane == 0) red[wave] = least;
  __syncthreads();
  for (uint32_t w = 0; w < n_waves; w++) least = max(least, red[w]);
  // what reaches the highest bound; it stands at the front of its list
  auto gather = [&]() __attribute__((always_inline)) {
    auto put = [&](uint32_t place, uint32_t b, uint2 x, double v) __attribute__((always_inline)) {
      if (place < kPickList) ranks[place] = order64(v), rest[place] = make_uint3(b, x.x, x.y);
    };
    // entries j .. of list c of beam b, until one is below the bound
    auto follow = [&](uint32_t b, uint32_t c, uint32_t j) __attribute__((always_inline)) {
      for (; j < P.n_out; j++) {
        const uint2 x = lists[static_cast<size_t>(b) * per_beam + c * P.n_out + j];
        const double v = rank_of(b, x.x);
        if (x.x == 0 || order32(static_cast<float>(v)) < least) break;
        put(atomicAdd(&n_list, 1u), b, x, v);
      }
    };
    uint32_t n = 0;
#pragma unroll
    for (uint32_t j = 0; j < kHead; j++) n += my_first[j] >= least;
    if (n) {
      const uint32_t place = atomicAdd(&n_list, n);
#pragma unroll
      for (uint32_t j = 0; j < kHead; j++)
        if (j < n) put(place + j, wave, mine[j], my_value[j]);
      if (n == kHead && state[wave] == kOpen) follow(wave, lane, kHead);
    }
    for (uint32_t b = wave; b < P.n_beams; b += n_waves) {  // lists behind a lane's first one
      if (state[b] == kEnded && b != wave && lane == 0) {
        const double v = rank_of(b, 1);
        if (order32(static_cast<float>(v)) >= least) put(atomicAdd(&n_list, 1u), b, make_uint2(1, P.end_token), v);
      }
      if (state[b] != kOpen) continue;
      for (uint32_t c = lane + (b == wave ? 64 : 0); c < P.n_chunks; c += 64) follow(b, c, 0);
    }
    __syncthreads();
  };
  gather();
  if (n_list > kPickFew) {
    // a closer bound, halved on by counting each lane's first few entries
    uint32_t up = 0xFFFFFFFFu, n_least = 0xFFFFFFFFu;
    while (n_least > P.n_out + P.n_out / 2 && up - least > 1) {
      const uint32_t mid = least + (up - least) / 2;
      uint32_t n = 0;
#pragma unroll
      for (uint32_t j = 0; j < kHead; j++) n += __builtin_popcountll(__ballot(my_first[j] >= mid));
      __syncthreads();
      if (lane == 0) red[wave] = n;
      __syncthreads();
      n = 0;
      for (uint32_t w = 0; w < n_waves; w++) n += red[w];
      if (n >= P.n_out) least = mid, n_least = n; else up = mid;
    }
    __syncthreads();
    for (uint32_t i = t; i < kPickList + 8; i += threads) ranks[i] = 0;
    if (t == 0) n_list = 0;
    __syncthreads();
    gather();
  }
  const uint32_t c = n_list;
  if (c <= kPickList) {  // the place of each is the number of those before it
    for (uint32_t i = t; i < c; i += threads) {
      const unsigned long long r = ranks[i];
      const uint3 y = rest[i];
      const Cand k{r, y.x, y.y, y.z};
      uint32_t place = 0, same = 0;
      for (uint32_t j = 0; j < c; j += 8)
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) {
          const unsigned long long o = ranks[j + u];  // 0 behind the last
          place += o > r;
          same += o == r;
        }
      if (same > 1)
        for (uint32_t j = 0; j < c; j++) {
          const uint3 z = rest[j];
          if (ranks[j] == r) place += before(Cand{r, z.x, z.y, z.z}, k);
        }
      if (place < P.n_out) chosen[place] = k;
    }
  } else {  // too many that are equal, or nearly: the first one behind the last, n_out times
    Cand last{~0ull, 0, 0, 0};
    for (uint32_t i = 0; i < P.n_out; i++) {
      Cand first{0, 0, 0, kNoToken};
      for (uint32_t e = t; e < P.n_beams * per_beam; e += threads) {
        const uint32_t b = e / per_beam;
        if (state[b] == kGone || (state[b] == kEnded && e % per_beam != 0)) continue;
        const uint2 x = state[b] == kEnded ? make_uint2(1, P.end_token) : lists[e];
        if (x.x == 0) continue;
        const Cand k{order64(rank_of(b, x.x)), b, x.x, x.y};
        if (before(last, k) && (first.rank == 0 || before(k, first))) first = k;
      }
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) {
        const Cand o{__shfl_xor(first.rank, off, 64), __shfl_xor(first.beam, off, 64), __shfl_xor(first.logit, off, 64),
                     __shfl_xor(first.token, off, 64)};
        if (o.rank && (first.rank == 0 || before(o, first))) first = o;
      }
      if (lane == 0) best[wave] = first;
      __syncthreads();
      for (uint32_t w = 0; w < n_waves; w++) {
        const Cand o = best[w];
        if (o.rank && (first.rank == 0 || before(o, first))) first = o;
      }
      __syncthreads();
      if (t == 0) chosen[i] = first;
      last = first;
      if (first.rank == 0) break;
    }
  }
  __syncthreads();
  if (t < P.n_out) {  // all that an output may overwrite has been read
    const Cand k = chosen[t];
    const uint32_t o = s * P.n_out + t, b = k.rank ? k.beam : min(t, P.n_beams - 1);
    float v = -INFINITY;
    if (k.rank) v = static_cast<float>(state[b] == kEnded ? score[b] : score[b] + (static_cast<double>(value32(k.logit)) - lse[b]));
    P.scores_out[o] = v;
    P.tokens[o] = k.token;
    P.parents[o] = b;
    if (P.counts_out) P.counts_out[o] = k.rank ? count_in[b] + (state[b] == kOpen) : 0u;
    if (P.len_out) P.len_out[o] = len_in[b] + 1;
    if (t < wh::kMaxBeams) from[t] = b, have[t] = len_in[b];
  }
  if (!P.history) return;
  // A wave has a beam (or two), and 256 columns of the histories at a time: what the beams take
  // of them is read before any of it is written.
  constexpr uint32_t kColumns = 4, kBeams = (wh::kMaxBeams + kPickWaves - 1) / kPickWaves;
  __syncthreads();
  uint32_t most = 0;
  for (uint32_t i = 0; i < P.n_beams; i++) most = max(most, have[i]);
  const size_t end = min(static_cast<size_t>(most) + 1, P.history_stride);
  uint32_t* const h = P.history + static_cast<size_t>(row0) * P.history_stride;
  for (size_t p0 = 0; p0 < end; p0 += 64 * kColumns) {
    uint32_t v[kBeams][kColumns];
    bool moves[kBeams][kColumns];
#pragma unroll
    for (uint32_t u = 0; u < kBeams; u++) {
      const uint32_t i = min(wave + u * n_waves, P.n_beams - 1), parent = from[i], n = have[i], token = chosen[i].token;
#pragma unroll
      for (uint32_t j = 0; j < kColumns; j++) {
        const size_t p = p0 + 64 * j + lane;
        moves[u][j] = wave + u * n_waves < P.n_beams && p < end && (p == n || (p < n && parent != i));
        uint32_t old = 0;
        if (moves[u][j] && p < n) old = h[parent * P.history_stride + p];
        v[u][j] = p == n ? token : old;
      }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < kBeams; u++)
#pragma unroll
      for (uint32_t j = 0; j < kColumns; j++)
        if (moves[u][j]) h[static_cast<size_t>(wave + u * n_waves) * P.history_stride + p0 + 64 * j + lane] = v[u][j];
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
    asm volatile("" ::: "memory");  // the table stays in LDS: in registers it would cost waves
#pragma unroll
    for (int i = 0; i < NB; i++)
      if (c < n[i]) v[i] = base[from[i] + c];
#pragma unroll
    for (int i = 0; i < NB; i++)
      if (c < n[i])  // past the caches: 115 -> 105 us a call for 262 MB in a graph, 7.3 -> 6.4 for 16
        __builtin_nontemporal_store(v[i], &base[i * beam + c]);
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
  const size_t waves = r.n_beams < 4 ? 4 : r.n_beams < kPickWaves ? r.n_beams : kPickWaves;
  beam_pick_kernel<<<static_cast<unsigned>(n_seqs), static_cast<unsigned>(64 * waves), 0, s>>>(P);
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
