// tree_attention.hip -- grouped-query attention of a tree of drafted tokens
// over an f16 KV cache, with rotary position embedding, on gfx950.
//
// One step verifies n_tree drafted tokens ("nodes") of each of n_seqs
// sequences.  With A(t) the node t and its ancestors, p_t = ctx_len + |A(t)| - 1
// its position, and G = n_heads / n_kv_heads:
//   q, k rotated as in attention.hip: pairs (i, i + d/2) by p_t * inv_freq[i]
//   cache row ctx_len + t = f16(k), f16(v)
//   s_j   = (q . k_j) / sqrt(d)   for j < ctx_len and j = ctx_len + a, a in A(t)
//   out_t = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m},  m = max_j s_j
// Three launches (two where the caches are short):
//   1. prepare: a wave per two heads of a node rotates q into f16 hi + lo limbs,
//      stores k and v in the cache and writes the node's ancestor mask; one more
//      workgroup cuts the sequences into chunks of equal length
//   2. partial: one workgroup per (chunk, KV head, group of 32 RW query rows)
//   3. combine: one workgroup per 32 query rows and 8 dims joins their chunks
//
// What bounds it.  Short and middle contexts: the launches' dependent loads and
// their ends.  26 nodes at 4070 positions, 32 / 8 heads of 128 (17.8 MB: 3.7 us at
// the 4.8 TB/s of a large copy): 4.2 + 14.2 + 4.0 us, of the partial kernel's 14.2
// some 3 until the first data is there, 6 for 4 tiles a wave, 2 for writing 6.9 MB of
// partial results.  8 sequences of 16 nodes up to 8100, 32 / 4 heads of 64: 4.9 + 12.9
// + 4.2.  5 nodes at 300 of 312 rows: 3.6 + 10.7.  Long contexts: the matrix cores.  64
// nodes at 131000: 275 GFLOP of limb products in 252 us, 1.1 PFLOP/s; a large f16
// library product reaches 1.15 on this card, where the clock falls under such work
// (467 k cycles, 56 % of them with a product under way).
//
// The angle is formed and reduced in 64 bits: in 32 bits p_t * inv_freq is off
// by up to p_t 2^-24 radians, 0.008 at position 131072.  k is rotated in
// 64 bits before its two roundings (to f32, to f16), so the stored row is the
// one the formula gives.
//
// Products on the matrix cores (v_mfma_f32_32x32x16_f16).  Rows of the query
// tile are (node, head of the group): r = t G + g.  S^T = K Q^T has lane l hold
// row l % 32 and 16 of the tile's 32 keys, so the softmax of a row needs one
// exchange with lane l ^ 32; the same registers, in the same key order, are
// the B operand of O^T = V^T P^T, whose A operand comes from the row-major V
// tile in LDS through transposing reads (ds_read_b64_tr_b16).  q is scaled by a
// power of two per row and split into f16 hi + lo, and so is P (e^{s - m} 2^12),
// with K and V taken from the cache as they are.  An element of q keeps 2^-22 of
// itself or 2^-38 of its row's largest.  P ends at 2^-25, so m follows the tiles'
// maxima, up and down: a weight keeps 2^-22 of itself or 2^-24 of its tile's largest.
// Beside one key with nearly all the weight (often the first, whose v is small, so
// that the others make the output) they keep what f32 would leave them; in that key's own
// tile they take a turn of their own.  Relative L2 with 90 to 99.9999 % of the weight on
// one key, up to 130000 positions: 3e-7 to 4e-6, the decode step's 5e-7 to 3e-6 (with m
// the running maximum alone 1e-5 to 0.2).
#include <type_traits>

#include "gemm_dev.hpp"
#include "tree.hpp"

namespace {

constexpr int kPrepThreads = 256;
constexpr int kAttnWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
// Weights are held in f16 as 2^12 e^{s - m}, hi + lo.  The reference m of a row stays
// where it is while the weight of a tile's largest score is within [2^-13, 2^3] of it (at
// most 2^15 in f16), else it moves there, up or down, but never 2^48 below its highest.
// Scores of deviation 1.3 move some row's in 3 % of the tiles, of 3 in 8 to 12 %: 64 nodes
// at 131000 positions take 280 and 284 us a call.
constexpr float kPScaleLog2 = 12.0f, kMoveUp = 3.0f, kMoveDown = -13.0f, kLowest = 48.0f;
// A row's keys in a tile are four groups, by their parity and by the lane that holds
// them.  Where the largest weight of a group is below 2^-22 of the reference's (2^-10 in
// f16: off by 2^-15 of itself), the row moves to the tile's maximum, and where it is so
// against that too, the tile takes two turns: the keys down to 2^-9 of its largest weight,
// then the others.  Scores of deviation 3 never do, of 5 in 3 % of the tiles of 64 keys and in
// 13 % of those of 32 (323 us).
constexpr float kFaint = -22.0f, kNear = 9.0f;
constexpr int kWholeMask = 4;        // mask words per node

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // four floats of the caller's output
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct Params {
  const float *q, *k, *v;
  size_t ldq, ldkv;
  const int32_t* parents;
  const uint32_t* ctx_len;
  _Float16 *k_cache, *v_cache;
  const float* inv_freq;
  float* out;
  uint32_t n_seqs, n_tree, max_ctx, n_heads, n_kv, G, R, n_rg, max_slots, target, sparse, lone, unit, least, tiles;
  float scale;
  // workspace
  uint4* slots;         // [max_slots] (sequence | rows of its tree << 16, first key, key behind the last, cache rows of the
                        // step); sequence n_seqs: none
  uint32_t* first;      // [n_seqs + 1] first slot
  uint32_t* mask;       // [n_seqs][n_tree][4]
  float* qscale;        // [n_seqs][n_kv][R]
  _Float16* qlimb;      // [n_seqs][n_kv][R][2][D]
  // partial results of a slot, KV head and tile of 32 query rows
  float2* ml;           // [max_slots][n_kv][tiles][32] (reference, sum)
  float4* acc;          // [max_slots][n_kv][tiles][D / 8][64]: the registers of the lanes, as in the product
};

// ------------------------------------------------------------------ prepare
// A 64-bit value as the cache holds it: rounded to f32, then to f16.  (The
// empty statement keeps the compiler from joining the two into one rounding.)
__device__ __forceinline__ _Float16 stored(double x) {
  float f = static_cast<float>(x);
  asm("" : "+v"(f));
  return static_cast<_Float16>(f);
}

// n: the rows that the tree takes (tree_rows)
__device__ __forceinline__ bool seq_fits(const Params& P, uint32_t ctx, uint32_t n) {
  return ctx <= P.max_ctx && n <= P.max_ctx - ctx;
}

// Inclusive prefix sum over the workgroup's 256 threads, and their total; red: 4
// words of LDS.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* red, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t up = __shfl_up(v, off, 64);
    if (lane >= off) v += up;
  }
  whd::lds_barrier();
  if (lane == 63) red[wave] = v;
  whd::lds_barrier();
  const uint32_t a = red[0], b = red[1], c = red[2], d = red[3];
  total = a + b + c + d;
  return v + (wave > 0 ? a : 0) + (wave > 1 ? b : 0) + (wave > 2 ? c : 0);
}

// Cuts the sequences into chunks of one length, a multiple of a stage of the
// partial kernel, so long and short sequences share the workgroups evenly
// whatever the lengths on the device.  About `target` chunks over all sequences
// give every CU two workgroups, whose matrix and vector work overlap; while theirs
// would have up to `lone` keys, `sparse` chunks, one workgroup per CU, do: half the
// partial results to write and to join.  (32 / 8 heads of 128, 26 nodes at 18000
// and 25000 positions, lone = 1024 against 512 and then chunks of 512: 34.3 / 40.5,
// 41.0 / 46.0 us; at 31000 53.0 / 53.1.)
// Thread t plans sequences [t per, (t + 1) per); first, nodes, ends (cache rows of the
// step, 0 for a sequence without work): LDS [n_seqs].  All rows together number less
// than 2^32 (checked by the host).
constexpr uint32_t kDeepChunk = 512;
__device__ void plan_chunks(const Params& P, uint32_t* first, uint32_t* nodes, uint32_t* ends, uint32_t* red) {
  const uint32_t t = threadIdx.x;
  const uint32_t per = (P.n_seqs + kPrepThreads - 1) / kPrepThreads;
  const uint32_t s0 = min(t * per, P.n_seqs), s1 = min(s0 + per, P.n_seqs);
  const uint32_t ctx0 = s0 < s1 ? P.ctx_len[s0] : 0;  // asked for with the trees
  // the trees' rows (tree_rows): a wave looks at 4 times 64 / g trees at once, a lane at
  // one node of each (two where a tree has more than 64)
  const uint32_t g = P.n_tree > 32 ? 64 : P.n_tree > 1 ? 1u << (32 - __builtin_clz(P.n_tree - 1)) : 1;
  const uint32_t step = kPrepThreads / g;
  const int i = t & (g - 1), n_tree = P.n_tree;
  for (uint32_t s2 = __builtin_amdgcn_readfirstlane(t / 64) * (64 / g); s2 < P.n_seqs; s2 += 4 * step) {
    int a[4], b[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint32_t s = s2 + u * step + (t & 63) / g;
      const int32_t* parents = P.parents + static_cast<size_t>(s) * P.n_tree;
      a[u] = s < P.n_seqs && i < n_tree ? parents[i] : -2;
      b[u] = s < P.n_seqs && i + 64 < n_tree ? parents[i + 64] : -2;
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const uint32_t s = s2 + u * step + (t & 63) / g;
      const unsigned long long lo = __ballot(a[u] >= -1 && a[u] < i) >> (t & 63 & ~(g - 1)) & (~0ull >> (64 - g));
      const unsigned long long hi = __ballot(b[u] >= -1 && b[u] < i + 64);  // g is 64 where there are any
      if (i == 0 && s < P.n_seqs) nodes[s] = hi ? 128 - __builtin_clzll(hi) : lo ? 64 - __builtin_clzll(lo) : 0;
    }
  }
  whd::lds_barrier();
  uint32_t mine = 0;
  for (uint32_t s = s0; s < s1; s++) {
    const uint32_t ctx = s == s0 ? ctx0 : P.ctx_len[s];
    const uint32_t n = nodes[s] && seq_fits(P, ctx, nodes[s]) ? ctx + nodes[s] : 0;
    ends[s] = n;
    mine += n;
  }
  uint32_t total, used;
  block_scan(mine, red, total);
  uint32_t even = (total + P.target - 1) / P.target;
  const uint32_t lone = (total + P.sparse - 1) / P.sparse;
  even = lone <= P.lone ? lone : max(even, kDeepChunk);
  const uint32_t chunk = max((even + P.unit - 1) / P.unit * P.unit, P.least);
  uint32_t n = 0;
  for (uint32_t s = s0; s < s1; s++) n += (ends[s] + chunk - 1) / chunk;
  uint32_t at = block_scan(n, red, used) - n;
  for (uint32_t s = s0; s < s1; s++) {
    const uint32_t c = (ends[s] + chunk - 1) / chunk;
    first[s] = at;
    P.first[s] = at;
    at += c;
  }
  if (t == 0) P.first[P.n_seqs] = used;
  whd::lds_barrier();
  for (uint32_t y = t; y < P.max_slots; y += kPrepThreads) {
    uint32_t lo = 0, hi = P.n_seqs;  // the last sequence whose first slot is at most y
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (first[mid] <= y) lo = mid; else hi = mid;
    }
    uint4 slot = make_uint4(P.n_seqs, 0, 0, 0);
    if (y < used) {
      const uint32_t rows = ends[lo], c0 = (y - first[lo]) * chunk;
      slot = make_uint4(lo | nodes[lo] << 16, c0, min(c0 + chunk, rows), rows);
    }
    P.slots[y] = slot;
  }
}

// grid: (n_seqs * n_tree) nodes x n_groups groups of 4 N heads (the q heads, then
// the KV heads), then one workgroup for the chunks.  A wave takes N heads and asks
// for their rows before it looks at the tree.  With few nodes N = 2: the launch is
// as long as its dependent loads; with many N = 8, which share the walk and the
// angles (22 sequences of 81 nodes, 80 + 16 heads: 68 -> 37 us).
template <int D, int N>
__global__ __launch_bounds__(kPrepThreads) void tree_prepare_kernel(const Params P, uint32_t n_groups) {
  __shared__ uint32_t first[wh::kMaxTreeSeqs], nodes[wh::kMaxTreeSeqs], ends[wh::kMaxTreeSeqs];
  __shared__ uint32_t red[kPrepThreads / 64];
  if (blockIdx.x == P.n_seqs * P.n_tree * n_groups) {
    plan_chunks(P, first, nodes, ends, red);
    return;
  }
  const uint32_t group = blockIdx.x % n_groups, row_id = blockIdx.x / n_groups;
  const uint32_t s = row_id / P.n_tree, t = row_id % P.n_tree;
  const size_t row = row_id;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t i = lane % (D / 2);
  const uint32_t h0 = (group * (kPrepThreads / 64) + wave) * N, n_slots = P.n_heads + P.n_kv;
  float x[N], y[N], vx[N] = {}, vy[N] = {};
#pragma unroll
  for (int u = 0; u < N; u++) {
    const uint32_t hh = min(h0 + u, n_slots - 1);
    const bool is_q = hh < P.n_heads;
    const float* src = is_q ? P.q + row * P.ldq + static_cast<size_t>(hh) * D
                            : P.k + row * P.ldkv + static_cast<size_t>(hh - P.n_heads) * D;
    x[u] = src[i];
    y[u] = src[i + D / 2];
    if (!is_q) {
      const float* v = P.v + row * P.ldkv + static_cast<size_t>(hh - P.n_heads) * D;
      vx[u] = v[i];
      vy[u] = v[i + D / 2];
    }
  }
  const whd::TreeLanes tree = whd::tree_lanes(P.parents + static_cast<size_t>(s) * P.n_tree, P.n_tree);
  const float inv = P.inv_freq[i];
  const uint32_t ctx = P.ctx_len[s];
  const whd::TreePath path = whd::tree_path(tree, t);
  const bool fits = seq_fits(P, ctx, whd::tree_rows(tree)), present = path.present() && fits;
  if (group == 0 && tid < kWholeMask) {
    const unsigned long long w = (tid < 2 ? path.lo : path.hi) >> (32 * (tid & 1));
    P.mask[row * kWholeMask + tid] = present ? static_cast<uint32_t>(w) : 0u;
  }
  const double angle = static_cast<double>(ctx + path.depth) * static_cast<double>(inv);
  // q: the angle in turns, whole turns dropped in 64 bits
  const double turns = angle * 0.15915494309189535;
  float qsn, qcs;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), &qsn, &qcs);
  double sn = 0, cs = 0;
  if (h0 + N > P.n_heads) sincos(angle, &sn, &cs);
#pragma unroll
  for (int u = 0; u < N; u++) {
    const uint32_t hh = h0 + u;
    if (hh >= n_slots) break;
    if (hh < P.n_heads) {
      if (!present && lane < D / 2) {
        // an absent node's rows are zeros; those of a sequence that does not fit its cache are NaN
        const float fill = fits ? 0.f : __builtin_nanf("");
        float* o = P.out + row * P.n_heads * D + static_cast<size_t>(hh) * D;
        o[i] = fill;
        o[i + D / 2] = fill;
      }
      float a = present ? x[u] * qcs - y[u] * qsn : 0.f, b = present ? x[u] * qsn + y[u] * qcs : 0.f;
      const float mx = whd::wave_max(fmaxf(fabsf(a), fabsf(b)));
      // the row's largest magnitude to [2^13, 2^14): hi + lo hold every element
      // to 2^-22 of itself or 2^-38 of the largest
      int e = 0;
      if (mx > 0.f && mx < INFINITY) e = min(13 - ilogbf(mx), 100);
      a = ldexpf(a, e);
      b = ldexpf(b, e);
      const size_t qrow = (static_cast<size_t>(s) * P.n_kv + hh / P.G) * P.R + t * P.G + hh % P.G;
      _Float16* o = P.qlimb + qrow * 2 * D;
      if (lane < D / 2) {
        const _Float16 ah = static_cast<_Float16>(a), bh = static_cast<_Float16>(b);
        o[i] = ah;
        o[i + D / 2] = bh;
        o[D + i] = static_cast<_Float16>(a - static_cast<float>(ah));
        o[D + i + D / 2] = static_cast<_Float16>(b - static_cast<float>(bh));
      }
      if (lane == 0) P.qscale[qrow] = ldexpf(P.scale * kLog2e, -e);
    } else if (present && lane < D / 2) {
      // k and v into the cache row of the node
      const size_t at = ((static_cast<size_t>(s) * P.max_ctx + ctx + t) * P.n_kv + (hh - P.n_heads)) * D;
      P.k_cache[at + i] = stored(x[u] * cs - y[u] * sn);
      P.k_cache[at + i + D / 2] = stored(x[u] * sn + y[u] * cs);
      P.v_cache[at + i] = static_cast<_Float16>(vx[u]);
      P.v_cache[at + i + D / 2] = static_cast<_Float16>(vy[u]);
    }
  }
}

// ------------------------------------------------------------------ partial
// LDS rows of K and V are D f16 without padding (the copies write 16 lanes'
// chunks in a row), so the 16-byte chunks of row r are permuted: chunk c lies
// at c ^ swz(r).  K: a wave's operand read takes one chunk of 32 rows; V: a
// transposing read takes four chunks of each of 4 rows.  With these every 16
// (32) lanes reach all 64 banks once.
template <int D>
__device__ __forceinline__ int swz_k(int r) { return D == 128 ? (r & 15) : ((r >> 1) & 7); }
template <int D>
__device__ __forceinline__ int swz_v(int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }

__device__ __forceinline__ s16x4 read_tr(uint32_t lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)lds);
}

// The largest of this lane's and lane ^ 32's value: NaN passed over, or kept.
__device__ __forceinline__ float swap_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float swap_max_nan(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_elementwise_maximum(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
                                       __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ __forceinline__ float swap_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_bit_cast(float, static_cast<uint32_t>(r[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(r[1]));
}

// The f16 values of a fragment with infinities and NaN replaced by 0.
__device__ __forceinline__ half8 finite_only(half8 x) {
  u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if ((w[i] & 0x7C00u) == 0x7C00u) w[i] &= 0xFFFF0000u;
    if ((w[i] & 0x7C000000u) == 0x7C000000u) w[i] &= 0x0000FFFFu;
  }
  return __builtin_bit_cast(half8, w);
}

// Replaces the infinities and NaN of a 32-row V tile in LDS by 0 and tells
// whether there were any: lane l looks through half of row l / 2 (the order of
// its chunks does not matter).  Waves that share a tile may do so at the same
// time: they store the same values, each before it reads the tile itself.  But
// one that looks after another has stored finds nothing: only all of them
// together know what the tile held.
template <int D>
__device__ __forceinline__ bool clean_tile(uint32_t vt, int lane) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  auto at = [&](int j) { return reinterpret_cast<__attribute__((address_space(3))) u32x4*>((uintptr_t)(vt + lane * D + 16 * j)); };
  u16x2 top = {0, 0};  // the largest exponent of the even and of the odd elements
#pragma unroll
  for (int j = 0; j < D / 16; j++) {
    const u32x4 w = *at(j);
#pragma unroll
    for (int i = 0; i < 4; i++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7C007C00u));
  }
  const bool bad = top[0] == 0x7C00 || top[1] == 0x7C00;
  if (!__ballot(bad)) return false;
#pragma unroll 1
  for (int j = 0; j < D / 16; j++) *at(j) = __builtin_bit_cast(u32x4, finite_only(__builtin_bit_cast(half8, *at(j))));
  return true;
}

// Two weights as f16 hi + lo: elements i and i + 1 of the fragments.  hi is
// rounded to nearest, lo is what it leaves (one v_fma_mix each).
__device__ __forceinline__ void split2(float a, float b, half8& hi, half8& lo, int i) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const half2v h = __builtin_convertvector((f32x2{a, b}), half2v);
  const uint32_t hw = __builtin_bit_cast(uint32_t, h);
  float ra, rb;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hw), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hw), "v"(b));
  const half2v r = __builtin_convertvector((f32x2{ra, rb}), half2v);
  hi[i] = h[0], hi[i + 1] = h[1];
  lo[i] = r[0], lo[i + 1] = r[1];
}

// RW query tiles of 32 rows per workgroup; the 4 waves are RW rows x KW keys.
template <int D, int RW>
struct Shape {
  static constexpr int KW = kAttnWaves / RW;
  static constexpr int SK = KW == 4 ? 128 : 64;              // keys per stage
  static constexpr int TILES = SK / 32 / KW;                 // 32-key tiles per wave and stage
  static constexpr int kTileBytes = SK * D * 2;              // one of K, V
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kMergeBytes = KW > 1 ? kAttnWaves * 32 * (D + 2) * 4 : 0;  // all waves' sums, maxima and totals
  static constexpr int kFlag = 2 * kStageBytes > kMergeBytes ? 2 * kStageBytes : kMergeBytes;  // a word: a tile was cleaned
  static constexpr int kLds = kFlag + 16;
};

// grid: n_kv * n_rg * max_slots, KV head fastest (with 8 KV heads the workgroups
// of one head run on one XCD and share its L2).
template <int D, int RW>
__global__ __launch_bounds__(64 * kAttnWaves, RW == 1 && D == 128 ? 1 : 2) void tree_partial_kernel(const Params P) {
  using S = Shape<D, RW>;
  constexpr int KW = S::KW, SK = S::SK, DT = D / 32, KS = D / 16;
  extern __shared__ __align__(256) unsigned char lds[];
  const uint32_t kvh = blockIdx.x % P.n_kv, rg = blockIdx.x / P.n_kv % P.n_rg, slot = blockIdx.x / (P.n_kv * P.n_rg);
  const uint4 sc = P.slots[slot];
  const uint32_t seq = sc.x & 0xFFFFu, c0 = sc.y, c1 = sc.z, rows = sc.w;  // c0 < c1 <= rows
  if (seq >= P.n_seqs) return;
  const uint32_t ctx = rows - (sc.x >> 16);
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave / KW, kw = wave % KW;
  const size_t RS = static_cast<size_t>(P.n_kv) * D * 2;  // bytes between cache rows
  const size_t head0 = (static_cast<size_t>(seq) * P.max_ctx * P.n_kv + kvh) * D * 2;
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(P.k_cache) + head0;
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(P.v_cache) + head0;
  const uint32_t lds0 = lds_addr(lds);

  // One stage: rows [k0, k0 + SK) of K and V; a wave copies 1 KB (1024 / (2 D)
  // rows) of each at a time, the workgroup kRowsAll rows.  The chunks'
  // permutation repeats within kRowsAll rows, so a lane's offset is the same
  // each time.  Rows past the last one repeat it: they are masked.
  constexpr int kRowsPer = 1024 / (2 * D), kRowsAll = kRowsPer * kAttnWaves, kChunks = D / 8;
  const int crow = wave * kRowsPer + lane / kChunks, cchunk = lane % kChunks;
  const uint32_t ck = 16 * (cchunk ^ swz_k<D>(crow)), cv = 16 * (cchunk ^ swz_v<D>(crow));
  const uint32_t crs = crow * static_cast<uint32_t>(RS);
  auto issue = [&](uint32_t k0, int buf) {
    const uint8_t* kb = kbase + k0 * RS;
    const uint8_t* vb = vbase + k0 * RS;
    uint32_t at = lds0 + buf * S::kStageBytes + wave * 1024;
    if (k0 + SK <= rows) {
#pragma unroll
      for (int j = 0; j < SK / kRowsAll; j++) {
        copy16_to_lds(kb, crs + ck, at);
        copy16_to_lds(vb, crs + cv, at + S::kTileBytes);
        kb += kRowsAll * RS;
        vb += kRowsAll * RS;
        at += kAttnWaves * 1024;
      }
    } else {
      const uint32_t last = rows - 1 - k0;
#pragma unroll
      for (int j = 0; j < SK / kRowsAll; j++) {
        const uint32_t row = min(static_cast<uint32_t>(crow + kRowsAll * j), last) * static_cast<uint32_t>(RS);
        copy16_to_lds(kb, row + ck, at);
        copy16_to_lds(vb, row + cv, at + S::kTileBytes);
        at += kAttnWaves * 1024;
      }
    }
  };
  issue(c0, 0);

  // this wave's query rows
  const uint32_t r0 = (rg * RW + rw) * 32 + l32;
  const uint32_t r = min(r0, P.R - 1);
  const size_t qrow = (static_cast<size_t>(seq) * P.n_kv + kvh) * P.R + r;
  half8 qh[KS], ql[KS];
#pragma unroll
  for (int j = 0; j < KS; j++) {
    const _Float16* q = P.qlimb + qrow * 2 * D + 16 * j + 8 * h;
    qh[j] = *reinterpret_cast<const half8*>(q);
    ql[j] = *reinterpret_cast<const half8*>(q + D);
  }
  // scores are qs times s, in powers of 2; the reference m is kept as s, so that
  // the exponent of its key is exactly 0 however large it is
  const float qs = P.qscale[qrow];
  uint32_t tm[kWholeMask] = {};
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[d][i] = 0.f;
  // A lane's place in a K tile (row l32, chunk h; of step j chunk 2 j + h) and in a V
  // tile (row 4 h + kq, dims 16 dg + 4 dq ..; of 32 dims d chunk 4 d + ..).  The chunks'
  // permutations turn bits of the address, so steps and dims do as well.
  const int kq = (lane & 15) >> 2, dq = lane & 3, dg = (lane >> 4) & 1;
  const uint32_t ko = l32 * 2 * D + 16 * (h ^ swz_k<D>(l32));
  const uint32_t vo = (4 * h + kq) * 2 * D + 16 * ((2 * dg + (dq >> 1)) ^ swz_v<D>(kq)) + 8 * (dq & 1);
  float m = -INFINITY, floor = -INFINITY, l = 0.f;
  bool odd = false;  // V holds infinities or NaN
  uint32_t* const cleaned = reinterpret_cast<uint32_t*>(lds + S::kFlag);
  if (RW > 1 && tid == 0) *cleaned = 0;  // seen by all from the first stage's barrier on

  // N 32-key tiles, KW tiles apart.  kt, vt: LDS addresses of the first one's first
  // K and V row.  Edge (N = 1): the tile may reach beyond the cache into the nodes'
  // rows or past the last one.
  // Returns whether the tiles need a second turn, for the keys that the first left out.
  auto turn_of = [&](uint32_t base, uint32_t kt, uint32_t vt, auto edge, auto count, auto second) __attribute__((always_inline)) {
    constexpr bool kEdge = decltype(edge)::value;
    constexpr int N = decltype(count)::value, kStep = KW * 32 * 2 * D;
    constexpr bool kSecond = decltype(second)::value;
    f32x16 s[N];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < 16; i++) s[n][i] = 0.f;
    // LDS reads run one step ahead of the matrix products that take them: kNoLds
    // lets the compiler move anything but them across
    constexpr int kNoLds = 0x47F;
    half8 kf[2][N];
    auto k_at = [&](int j, int n) {
      return *reinterpret_cast<const __attribute__((address_space(3))) half8*>(
          (uintptr_t)(((kt + ko) ^ (32 * j)) + n * kStep));
    };
    auto read_k = [&](int j) {
#pragma unroll
      for (int n = 0; n < N; n++) kf[j & 1][n] = k_at(j, n);
      __builtin_amdgcn_sched_barrier(kNoLds);
    };
    read_k(0);
#pragma unroll
    for (int j = 0; j < KS; j++) {
      if (j + 1 < KS) read_k(j + 1);
#pragma unroll
      for (int n = 0; n < N; n++) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j & 1][n], qh[j], s[n], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < N; n++) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[j & 1][n], ql[j], s[n], 0, 0, 0);
    }
    if constexpr (kEdge) {
      static_assert(N == 1, "one tile at a time");
      uint32_t bits;
      // keys from ctx on are the tree's nodes: bit k of `bits` for key base + k
      const int off = static_cast<int>(base) - static_cast<int>(ctx);
      if (off <= -32) {
        bits = 0xFFFFFFFFu;
      } else if (off < 0) {
        bits = (tm[0] << -off) | ((1u << -off) - 1u);
      } else {
        const int w = off >> 5, sh = off & 31;
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int i = 0; i < kWholeMask; i++) {
          if (i == w) lo = tm[i];
          if (i == w + 1) hi = tm[i];
        }
        bits = sh ? (lo >> sh) | (hi << (32 - sh)) : lo;
      }
      if (clean_tile<D>(vt, lane)) {
        odd = true;
        if (RW > 1) *cleaned = 1;
      }
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int key = 8 * (i >> 2) + 4 * h + (i & 3);
        s[0][i] = (bits >> key) & 1u ? s[0][i] : -INFINITY;
      }
    }
    half8 vf[2][DT];
    auto read_v = [&](int ks) {
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const s16x4 x = read_tr(((vt + vo) ^ (64 * d)) + ks / 2 * kStep + (16 * (ks % 2) + 8 * u) * 2 * D);
          const auto y = __builtin_bit_cast(_Float16 __attribute__((ext_vector_type(4))), x);
#pragma unroll
          for (int i = 0; i < 4; i++) vf[ks & 1][d][4 * u + i] = y[i];
        }
      __builtin_amdgcn_sched_barrier(kNoLds);
    };
    read_v(0);
    // the largest score of each group of keys, and of the row
    float top[2], mt;
    auto tops = [&](auto larger) {
#pragma unroll
      for (int i = 0; i < 16 * N; i++) top[i & 1] = i < 2 ? s[0][i] : larger(top[i & 1], s[i / 16][i % 16]);
      mt = larger(top[0], top[1]);
    };
    tops([](float x, float y) { return __builtin_elementwise_maximum(x, y); });
    mt = swap_max_nan(mt);
    if (__builtin_expect(__ballot(mt != mt) != 0, 0)) {
      // A score is NaN: the formula's, or made of an infinity in K that q's limbs meet
      // with both signs or as 0.  q's sign and size are the hi limb's: its product alone
      // says what an infinity makes of the score (an element of q below 2^-38 of its
      // row's largest counts as 0 here).
#pragma unroll
      for (int n = 0; n < N; n++) {
        f32x16 x;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = 0.f;
#pragma unroll 1
        for (int j = 0; j < KS; j++) {
          half8 q = qh[0];
#pragma unroll
          for (int u = 1; u < KS; u++) q = j == u ? qh[u] : q;
          x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k_at(j, n), q, x, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (s[n][i] != s[n][i]) s[n][i] = x[i];
      }
      tops([](float x, float y) { return fmaxf(x, y); });
      mt = swap_max(mt);
      read_v(0);  // so that its registers are free above
    }
    if constexpr (kEdge) {
#pragma unroll
      for (int i = 0; i < 2; i++) top[i] = top[i] == -INFINITY ? INFINITY : top[i];  // masked keys are not faint
    }
    float low = fminf(top[0], top[1]);  // of the lane's two groups, then of the row's four
    const float far = (mt - m) * qs;
    bool again = false;
    if (kSecond || __ballot(far > kMoveUp || far < kMoveDown || (low - m) * qs < kFaint)) {
      low = -swap_max(-low);
      if (kSecond || __builtin_expect(__ballot((low - mt) * qs < kFaint) != 0, 0)) {
        // first the keys near the tiles' maximum, then the others, with a reference of their own
        const float split = mt - kNear * __builtin_amdgcn_rcpf(qs);
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
          for (int i = 0; i < 16; i++) s[n][i] = (s[n][i] < split) != kSecond ? -INFINITY : s[n][i];
        tops([](float x, float y) { return fmaxf(x, y); });
        mt = swap_max(mt);
        again = !kSecond;
      }
      const float to = mt == -INFINITY ? m : fmaxf(mt, floor);  // -inf: the row sees nothing here
      const float by = (to - m) * qs;
      const bool moves = by > kMoveUp || by < ((low - m) * qs < kFaint ? -kMoveUp : kMoveDown);
      const float al = moves ? __builtin_amdgcn_exp2f(-by) : 1.f;
      l *= al;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] *= al;
      if (moves) m = to, floor = fmaxf(floor, to - kLowest * __builtin_amdgcn_rcpf(qs));
    }
    const float mb = m == -INFINITY ? 0.f : m;
    float lt[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < 2 * N; ks++) {
      half8 ph, pl;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float p[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          p[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks / 2][8 * (ks % 2) + i + k] - mb, qs, kPScaleLog2));
          lt[(i + k) & 3] += p[k];
        }
        split2(p[0], p[1], ph, pl, i);
      }
      if (ks + 1 < 2 * N) read_v(ks + 1);
#pragma unroll
      for (int d = 0; d < DT; d++) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[ks & 1][d], ph, acc[d], 0, 0, 0);
#pragma unroll
      for (int d = 0; d < DT; d++) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[ks & 1][d], pl, acc[d], 0, 0, 0);
    }
    l += (lt[0] + lt[1]) + (lt[2] + lt[3]);  // one addition to the running sum
    return again;
  };

  auto tiles = [&](uint32_t base, uint32_t kt, uint32_t vt, auto edge, auto count) {
    if (__builtin_expect(turn_of(base, kt, vt, edge, count, std::false_type{}), 0))
      turn_of(base, kt, vt, edge, count, std::true_type{});
  };

  // stages of cache rows only, then those that reach the nodes' rows or the chunk's end
  const uint32_t n_stages = (c1 - c0 + SK - 1) / SK;
  const uint32_t inner = min(c1, ctx), n_inner = inner > c0 ? (inner - c0) / SK : 0;
  auto turn = [&](uint32_t st) {
    wait_vmcnt<0>();  // this wave's copies of stage st
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // everyone's; and everyone has read stage st - 1
    asm volatile("" ::: "memory");
    if (st + 1 < n_stages) issue(c0 + (st + 1) * SK, (st + 1) & 1);
    return lds0 + (st & 1) * S::kStageBytes;
  };
  uint32_t st = 0;
  for (; st < n_inner; st++) {
    const uint32_t kt = turn(st), to = 32 * kw * 2 * D;
    tiles(0, kt + to, kt + S::kTileBytes + to, std::false_type{}, std::integral_constant<int, S::TILES>{});
  }
  {
    const uint4 w = *reinterpret_cast<const uint4*>(P.mask + (static_cast<size_t>(seq) * P.n_tree + r / P.G) * kWholeMask);
    tm[0] = w.x, tm[1] = w.y, tm[2] = w.z, tm[3] = w.w;
  }
#pragma unroll 1
  for (; st < n_stages; st++) {
    const uint32_t kt = turn(st);
#pragma unroll 1
    for (int u = 0; u < S::TILES; u++) {
      const uint32_t base = c0 + st * SK + 32 * (kw + KW * u), to = 32 * (kw + KW * u) * 2 * D;
      if (base < c1) tiles(base, kt + to, kt + S::kTileBytes + to, std::true_type{}, std::integral_constant<int, 1>{});
    }
  }
  l = swap_sum(l);
  if constexpr (RW > 1) {
    whd::lds_barrier();
    odd = *cleaned != 0;  // waves of different rows share their tiles: one of them found what there was
  }
  // Infinities and NaN of V count for the query rows that see them, and for no
  // other.  The edge tiles took them out (0 * inf would have spread a NaN), in the
  // others they made infinities and NaN of these sums, of either kind (the lo limb
  // of a weight may be below 0).  Every weight is above 0, so such an element's
  // sum is that of the infinities and NaN alone: the rows are read again for them.
  {
    float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) zero[i & 3] = __builtin_fmaf(acc[d][i], 0.f, zero[i & 3]);
    odd |= __ballot(!((zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.f)) != 0;
  }
  if (odd) {
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (!(fabsf(acc[d][i]) < INFINITY)) acc[d][i] = 0.f;
    for (uint32_t base = c0 + 32 * kw; base < c1; base += 32 * KW) {
      // lane l looks through half of row l / 2
      const uint32_t look = min(base + lane / 2, c1 - 1);
      const uint4* half = reinterpret_cast<const uint4*>(vbase + look * RS + (lane & 1) * D);
      bool bad = false;
      for (int j = 0; j < D / 16; j++) {
        const uint4 w = half[j];
        for (const uint32_t x : {w.x, w.y, w.z, w.w}) bad |= (x & 0x7C00u) == 0x7C00u || (x & 0x7C000000u) == 0x7C000000u;
      }
      unsigned long long rows_bad = __ballot(bad);
      rows_bad = (rows_bad | rows_bad >> 1) & 0x5555555555555555ull;  // bit 2 k: row k
      while (rows_bad) {
        const uint32_t key = base + __builtin_ctzll(rows_bad) / 2;
        rows_bad &= rows_bad - 1;
        if (key >= c1) break;  // the last row, looked at again
        const uint32_t node = key - ctx;  // wraps for the cache's rows
        uint32_t w = tm[0];
#pragma unroll
        for (int i = 1; i < kWholeMask; i++)
          if (node >> 5 == static_cast<uint32_t>(i)) w = tm[i];
        if (key >= ctx && !((w >> (node & 31)) & 1u)) continue;
        const _Float16* v = reinterpret_cast<const _Float16*>(vbase + key * RS);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const float x = static_cast<float>(v[32 * d + 8 * (i >> 2) + 4 * h + (i & 3)]);
            if (!(fabsf(x) < INFINITY)) acc[d][i] += x;
          }
      }
    }
  }

  // A sequence in one chunk is done: its rows go to the caller's output.  Else
  // results go out in the lanes' own order: a wave stores 1 KB in a row, and the
  // combine kernel reads it back the same way.
  constexpr int kQuads = D / 8;  // float4 per lane
  const bool whole = c0 == 0 && c1 == rows;
  const size_t tile0 = (static_cast<size_t>(slot) * P.n_kv + kvh) * P.n_rg * RW + rg * RW;
  const uint32_t node = r / P.G;
  float* const orow = P.out + (static_cast<size_t>(seq) * P.n_tree + node) * P.n_heads * D +
                      static_cast<size_t>(kvh * P.G + r % P.G) * D + 4 * h;
  // a row to store: not one of the padding, nor, in the output, an absent node's
  const bool mine = r0 < P.R && (!whole || (tm[0] | tm[1] | tm[2] | tm[3]) != 0);
  auto put = [&](int q, float4 a, float total) {
    if (whole) *reinterpret_cast<f32x4u*>(orow + 32 * (q >> 2) + 8 * (q & 3)) = f32x4u{a.x, a.y, a.z, a.w} / total;
    else P.acc[((tile0 + rw) * kQuads + q) * 64 + lane] = a;
  };
  if constexpr (KW == 1) {
    if (mine) {
#pragma unroll
      for (int q = 0; q < kQuads; q++) {
        const f32x16& v = acc[q / 4];
        const int i = 4 * (q % 4);
        put(q, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]), l);
      }
      if (h == 0 && !whole) P.ml[(tile0 + rw) * 32 + l32] = make_float2(m, l);
    }
  } else {
    // the KW waves of each query tile join in LDS, in fixed order
    whd::lds_barrier();
    float4* am = reinterpret_cast<float4*>(lds);                       // [4][D / 8][64]
    float2* mm = reinterpret_cast<float2*>(am + kAttnWaves * kQuads * 64);  // [4][32]
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        am[(wave * kQuads + 4 * d + i) * 64 + lane] =
            make_float4(acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]);
    if (h == 0) mm[wave * 32 + l32] = make_float2(m, l);
    whd::lds_barrier();
    // wave -> its query tile's quads kw, kw + KW, ...
    float M = -INFINITY, L = 0.f, ew[KW];
    float2 ml[KW];
#pragma unroll
    for (int w = 0; w < KW; w++) {
      ml[w] = mm[(rw * KW + w) * 32 + l32];
      M = fmaxf(M, ml[w].x);
    }
#pragma unroll
    for (int w = 0; w < KW; w++) {
      ew[w] = ml[w].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[w].x - M) * qs);
      L = __builtin_fmaf(ml[w].y, ew[w], L);
    }
    if (mine) {
#pragma unroll
      for (int q = 0; q < kQuads / KW; q++) {
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KW; w++) {
          const float4 a = am[((rw * KW + w) * kQuads + kw + KW * q) * 64 + lane];
          A.x = __builtin_fmaf(a.x, ew[w], A.x);
          A.y = __builtin_fmaf(a.y, ew[w], A.y);
          A.z = __builtin_fmaf(a.z, ew[w], A.z);
          A.w = __builtin_fmaf(a.w, ew[w], A.w);
        }
        put(kw + KW * q, A, L);
      }
      if (kw == 0 && h == 0 && !whole) P.ml[(tile0 + rw) * 32 + l32] = make_float2(M, L);
    }
  }
}

// ------------------------------------------------------------------ combine
// out = sum_c acc_c w_c / sum_c l_c w_c, w_c = 2^{(m_c - M) qs}.  An item is one register
// quad of a tile of 32 query rows: lane l has four dims of row l % 32, so every
// row's maximum and sums stay in its lane, and a load is 1 KB in a row.  Wave w
// joins chunks w, w + W, .., 8 loads in flight, then the W waves join in fixed
// order.  Sequences in one chunk, and absent nodes, have their output.
// With few items W = 4 waves take one, with many W = 1 (a wave joins all chunks of
// its quad, and the workgroups stride over the items: 22 sequences
// of 81 nodes and 80 heads, most in one chunk: 28 -> 12 us).
// Items: n_kv x D / 8 quads x tiles x sequences, KV head fastest, as the partial
// kernel's workgroups: with 8 KV heads a head's chunks are joined on the XCD
// whose L2 they were written through.
template <int D, int W>
__global__ __launch_bounds__(256) void tree_combine_kernel(const Params P, uint32_t n_tiles, uint32_t n_items) {
  constexpr int kQuads = D / 8, kPer = 8, kGroup = 4 / W;  // quads per workgroup
  __shared__ float4 pa[W > 1 ? W : 1][64];
  __shared__ float2 pm[W > 1 ? W : 1][64];
  const uint32_t lane = threadIdx.x & 63, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t step = static_cast<size_t>(P.n_kv) * P.tiles;
  for (uint32_t item = blockIdx.x; item < n_items; item += gridDim.x) {
    uint32_t b = item;
    const uint32_t kvh = b % P.n_kv;
    b /= P.n_kv;
    const uint32_t quad = b % (kQuads / kGroup) * kGroup + wave / W;
    b /= kQuads / kGroup;
    const uint32_t tile = b % n_tiles, seq = b / n_tiles;
    const uint32_t row = tile * 32 + (lane & 31);
    const float qs = P.qscale[(static_cast<size_t>(seq) * P.n_kv + kvh) * P.R + min(row, P.R - 1)];
    const uint32_t c0 = P.first[seq], n = P.first[seq + 1] - c0;
    if (n <= 1) {
      if constexpr (W > 1) return;
      continue;
    }
    const size_t at = (static_cast<size_t>(c0) * P.n_kv + kvh) * P.tiles + tile;
    float M = -INFINITY, L = 0.f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    auto join = [&](float2 ml, float4 a) {
      // a part without a reference has no weight, but NaN of its scores stay
      const float ew = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - M) * qs);
      L = __builtin_fmaf(ml.y, ew, L);
      A.x = __builtin_fmaf(a.x, ew, A.x);
      A.y = __builtin_fmaf(a.y, ew, A.y);
      A.z = __builtin_fmaf(a.z, ew, A.z);
      A.w = __builtin_fmaf(a.w, ew, A.w);
    };
    for (uint32_t c = wave % W; c < n; c += W * kPer) {
      float2 ml[kPer];
      float4 a[kPer];
      float mx = M;
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        const size_t s = at + min(c + W * j, n - 1) * step;
        ml[j] = P.ml[s * 32 + (lane & 31)];
        a[j] = P.acc[(s * kQuads + quad) * 64 + lane];
      }
#pragma unroll
      for (int j = 0; j < kPer; j++)
        if (c + W * j < n) mx = fmaxf(mx, ml[j].x);
      const float keep = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((M - mx) * qs);
      M = mx;
      if (keep != 1.f) L *= keep, A.x *= keep, A.y *= keep, A.z *= keep, A.w *= keep;
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        if (c + W * j >= n) break;
        join(ml[j], a[j]);
      }
    }
    if constexpr (W > 1) {
      pa[wave][lane] = A;
      pm[wave][lane] = make_float2(M, L);
      whd::lds_barrier();
      if (wave == 0) {
        for (int w = 1; w < W; w++) M = fmaxf(M, pm[w][lane].x);
        L = 0.f;
        A = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < W; w++) join(pm[w][lane], pa[w][lane]);
      }
    }
    if ((W == 1 || wave == 0) && row < P.R) {
      const uint32_t t = row / P.G, g = row % P.G;
      const size_t node = static_cast<size_t>(seq) * P.n_tree + t;
      const uint4 w4 = *reinterpret_cast<const uint4*>(P.mask + node * kWholeMask);
      // no key's score above -inf: 0 / 0, as the formula
      if ((w4.x | w4.y | w4.z | w4.w) != 0)
        *reinterpret_cast<f32x4u*>(P.out + node * P.n_heads * D + static_cast<size_t>(kvh * P.G + g) * D +
                                   32 * (quad >> 2) + 8 * (quad & 3) + 4 * h) = f32x4u{A.x, A.y, A.z, A.w} / L;
    }
    if constexpr (W > 1) return;  // one item per workgroup
  }
}

// ------------------------------------------------------------------ launching
size_t al256(size_t v) { return (v + 255) / 256 * 256; }

// A cache of up to so many rows is one chunk: no partial results to join, no third
// launch.  A call, one chunk against several: 32 / 8 heads of 128, 5 nodes (20 query
// rows a KV head) at 300, 480 positions 13.2 / 15.4, 14.7 / 15.2 us, 100 sequences of
// them at 480 36.6 / 40.9; 26 nodes (104 rows) at 200, 360 13.1 / 15.3, 16.1 / 15.5; 32
// / 4 heads of 64, 10 nodes at 700 13.0 / 15.1, 64 nodes 15.6 / 15.8.  Workgroups of two
// or four tiles, whose waves have all keys to go through: 26 nodes at 120, 300 16.4 /
// 15.4, 20.7 / 15.7.
size_t single_rows(int rw, size_t R, size_t D) { return rw > 1 ? 128 : D == 64 ? 768 : R <= 32 ? 512 : 384; }

// Query tiles per workgroup: 1, 2 or 4.  With 4, K and V are read once per 128 rows;
// with fewer, the waves share the keys, and the workgroups that fill the CUs are a
// half or a quarter as many chunks, with as many fewer partial results.  So fewer are
// taken where the caches are short: one chunk a sequence with a tile per workgroup, or
// chunks of up to 384 (1 tile) or 512 keys (2 tiles), fill the CUs at most once.  A call with
// 32 / 8 heads of 128, fewer against 4 tiles: 26 nodes (104 query rows) at 200, 1000
// positions (1 tile) 13.1 / 16.2, 17.0 / 17.4 us, at 4070, 8100 (2) 20.3 / 22.1, 24.6 /
// 25.1, beyond at 16000 (2) 32.6 / 32.0; 64 nodes at 60 (1) 12.8 / 18.5, at 1000 (2)
// 20.2 / 21.3, beyond at 16000 (2) 49.1 / 48.3 and at 131000 292 / 276; 4 sequences of
// 40 nodes at 200, 4070 (1, 2) 16.2 / 19.6, 28.8 / 31.7.  (These, and the figures of
// single_rows and plan_chunks, were taken with m as the running maximum; a call of either
// form has taken 0 to 0.5 us more since.)
int row_tiles(size_t R, size_t D, size_t n_kv, size_t n_seqs, size_t max_ctx) {
  auto fits = [&](size_t rows, size_t keys) {
    const size_t chunks = n_seqs * ((max_ctx + keys - 1) / keys);
    return R <= rows || chunks * n_kv * ((R + rows - 1) / rows) <= static_cast<size_t>(wh::cu_count());
  };
  const size_t one = single_rows(1, R, D);
  return fits(32, 384) || (max_ctx <= one && fits(32, one)) ? 1 : fits(64, kDeepChunk) ? 2 : 4;
}

struct Plan {
  int rw;
  size_t G, R, n_rg, target, sparse, lone, unit, least, max_slots;
  bool single;  // every sequence is one chunk
};
Plan make_plan(size_t n_seqs, size_t n_tree, size_t n_heads, size_t n_kv, size_t D, size_t max_ctx) {
  Plan p;
  p.G = n_heads / n_kv;
  p.R = n_tree * p.G;
  p.rw = row_tiles(p.R, D, n_kv, n_seqs, max_ctx);
  p.n_rg = (p.R + 32 * p.rw - 1) / (32 * p.rw);
  p.unit = p.rw == 1 ? 128 : 64;
  // one workgroup per CU with 128 KB of stages, two with 64 KB; every sequence but
  // one may add a chunk by its rounding, and one workgroup too many is a second turn
  // (32 / 8 heads of 128, 4 sequences of 5 nodes at 20000 positions: 32.9 -> 29.4 us)
  const size_t per = n_kv * p.n_rg, cus = static_cast<size_t>(wh::cu_count());
  auto spread = [&](size_t wgs) {
    const size_t n = wgs / per ? wgs / per : 1;
    return n >= 4 * n_seqs ? n - (n_seqs - 1) : n;
  };
  p.sparse = spread(cus);
  // sequences that are many against the chunks leave CUs with one more or one less: 16
  // sequences of 16 nodes, 15000 positions in all, 33.7 us with 512, 35.4 with 1024
  p.lone = cus / per >= 4 * n_seqs ? 2 * kDeepChunk : kDeepChunk;
  p.target = spread((p.rw == 1 ? 1 : 2) * cus);
  p.single = max_ctx <= single_rows(p.rw, p.R, D);
  p.least = p.single ? (max_ctx + p.unit - 1) / p.unit * p.unit : p.unit;
  const size_t most = n_seqs * ((max_ctx + p.least - 1) / p.least);
  p.max_slots = p.target + n_seqs < most ? p.target + n_seqs : most;
  return p;
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
  const size_t slots = P.max_slots, rows = static_cast<size_t>(P.n_kv) * P.R;
  P.slots = reinterpret_cast<uint4*>(take(16 * slots));
  P.first = reinterpret_cast<uint32_t*>(take(4 * (static_cast<size_t>(P.n_seqs) + 1)));
  P.mask = reinterpret_cast<uint32_t*>(take(4 * kWholeMask * static_cast<size_t>(P.n_seqs) * P.n_tree));
  P.qscale = reinterpret_cast<float*>(take(4 * P.n_seqs * rows));
  P.qlimb = reinterpret_cast<_Float16*>(take(2 * 2 * D * P.n_seqs * rows));
  const size_t all_tiles = slots * P.n_kv * P.tiles;
  P.ml = reinterpret_cast<float2*>(take(8 * 32 * all_tiles));
  P.acc = reinterpret_cast<float4*>(take(4 * D * 32 * all_tiles));
  return off;
}

Params fill(const Plan& p, size_t n_seqs, size_t n_tree, size_t n_heads, size_t n_kv, size_t D, size_t max_ctx) {
  Params P{};
  P.n_seqs = static_cast<uint32_t>(n_seqs);
  P.n_tree = static_cast<uint32_t>(n_tree);
  P.max_ctx = static_cast<uint32_t>(max_ctx);
  P.n_heads = static_cast<uint32_t>(n_heads);
  P.n_kv = static_cast<uint32_t>(n_kv);
  P.G = static_cast<uint32_t>(p.G);
  P.R = static_cast<uint32_t>(p.R);
  P.n_rg = static_cast<uint32_t>(p.n_rg);
  P.max_slots = static_cast<uint32_t>(p.max_slots);
  P.target = static_cast<uint32_t>(p.target);
  P.sparse = static_cast<uint32_t>(p.sparse);
  P.lone = static_cast<uint32_t>(p.lone);
  P.unit = static_cast<uint32_t>(p.unit);
  P.least = static_cast<uint32_t>(p.least);
  P.tiles = static_cast<uint32_t>(p.n_rg * p.rw);
  P.scale = 1.0f / sqrtf(static_cast<float>(D));
  return P;
}

template <int D, int RW>
int launch_partial(const Params& P, hipStream_t s) {
  WH_ENSURE_LDS(static_cast<size_t>(Shape<D, RW>::kLds), &tree_partial_kernel<D, RW>);
  tree_partial_kernel<D, RW><<<P.n_kv * P.n_rg * P.max_slots, 64 * kAttnWaves, Shape<D, RW>::kLds, s>>>(P);
  WH_LAUNCH_CHECK("tree attention kernel launch");
  return WH_OK;
}

// Workgroups of 8 heads from which on 32 heads take one.
constexpr size_t kManyHeads = 4096;

template <int D>
int launch_all(const Params& P, const Plan& p, hipStream_t s) {
  const uint32_t nodes = P.n_seqs * P.n_tree, heads = P.n_heads + P.n_kv;
  if (static_cast<size_t>(nodes) * heads < 8 * kManyHeads) {
    const uint32_t n_groups = (heads + 7) / 8;
    tree_prepare_kernel<D, 2><<<nodes * n_groups + 1, kPrepThreads, 0, s>>>(P, n_groups);
  } else {
    const uint32_t n_groups = (heads + 31) / 32;
    tree_prepare_kernel<D, 8><<<nodes * n_groups + 1, kPrepThreads, 0, s>>>(P, n_groups);
  }
  WH_LAUNCH_CHECK("tree attention prepare launch");
  int st = p.rw == 1 ? launch_partial<D, 1>(P, s) : p.rw == 2 ? launch_partial<D, 2>(P, s) : launch_partial<D, 4>(P, s);
  if (st || p.single) return st;
  const uint32_t n_tiles = (P.R + 31) / 32;
  const size_t cus = static_cast<size_t>(wh::cu_count()), items = static_cast<size_t>(P.n_kv) * (D / 8) * n_tiles * P.n_seqs;
  if (items <= 8 * cus) {
    tree_combine_kernel<D, 4><<<static_cast<unsigned>(items), 256, 0, s>>>(P, n_tiles, static_cast<uint32_t>(items));
  } else {
    const size_t grid = items / 4 < 8 * cus ? items / 4 : 8 * cus;
    tree_combine_kernel<D, 1><<<static_cast<unsigned>(grid), 256, 0, s>>>(P, n_tiles, static_cast<uint32_t>(items / 4));
  }
  WH_LAUNCH_CHECK("tree attention combine launch");
  return WH_OK;
}

}  // namespace

namespace wh {

bool tree_attention_shape_ok(size_t n_heads, size_t n_kv_heads, size_t head_dim) {
  return (head_dim == 64 || head_dim == 128) && n_kv_heads > 0 && n_heads > 0 && n_heads <= 1024 && n_heads % n_kv_heads == 0;
}

size_t tree_attention_workspace_bytes(size_t n_seqs, size_t n_tree, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                                      size_t max_ctx) {
  const Plan p = make_plan(n_seqs, n_tree, n_heads, n_kv_heads, head_dim, max_ctx);
  Params P = fill(p, n_seqs, n_tree, n_heads, n_kv_heads, head_dim, max_ctx);
  return layout(P, head_dim, nullptr);
}

int launch_tree_attention(const TreeAttnArgs& a, void* workspace, hipStream_t s) {
  const Plan p = make_plan(a.n_seqs, a.n_tree, a.n_heads, a.n_kv_heads, a.head_dim, a.max_ctx);
  Params P = fill(p, a.n_seqs, a.n_tree, a.n_heads, a.n_kv_heads, a.head_dim, a.max_ctx);
  layout(P, a.head_dim, workspace);
  P.q = a.q, P.k = a.k, P.v = a.v;
  P.ldq = a.ldq, P.ldkv = a.ldkv;
  P.parents = a.parents;
  P.ctx_len = a.ctx_len;
  P.k_cache = static_cast<_Float16*>(a.k_cache);
  P.v_cache = static_cast<_Float16*>(a.v_cache);
  P.inv_freq = a.inv_freq;
  P.out = a.out;
  return a.head_dim == 128 ? launch_all<128>(P, p, s) : launch_all<64>(P, p, s);
}

}  // namespace wh

WH_API size_t wh_attention_tree_workspace_bytes(size_t n_seqs, size_t n_tree, size_t n_heads, size_t n_kv_heads,
                                                size_t head_dim, size_t max_ctx) {
  if (n_seqs == 0 || n_tree == 0 || max_ctx == 0 || n_seqs > wh::kMaxTreeSeqs || n_tree > wh::kMaxTreeNodes || max_ctx >> 31 ||
      n_seqs * max_ctx >> 32 ||
      !wh::tree_attention_shape_ok(n_heads, n_kv_heads, head_dim))
    return 0;
  return wh::tree_attention_workspace_bytes(n_seqs, n_tree, n_heads, n_kv_heads, head_dim, max_ctx);
}

WH_API int wh_attention_tree(const float* q, const float* k, const float* v, size_t ldq, size_t ldkv,
                             const int32_t* parents, const uint32_t* ctx_len, size_t n_seqs, size_t n_tree,
                             void* k_cache, void* v_cache, size_t max_ctx, size_t n_heads, size_t n_kv_heads,
                             size_t head_dim, const float* inv_freq, float* out, void* workspace,
                             size_t workspace_bytes, wh_stream_t stream) {
  if (!wh::tree_attention_shape_ok(n_heads, n_kv_heads, head_dim))
    return wh::set_error(WH_ERR_INVALID_SHAPE, "attention_tree: head_dim %zu, %zu heads, %zu KV heads not supported",
                         head_dim, n_heads, n_kv_heads);
  if (n_tree > wh::kMaxTreeNodes || n_seqs > wh::kMaxTreeSeqs)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "attention_tree: %zu nodes of %zu sequences (at most %zu of %zu)", n_tree,
                         n_seqs, wh::kMaxTreeNodes, wh::kMaxTreeSeqs);
  if (max_ctx == 0 || max_ctx >> 31)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "attention_tree: max_ctx = %zu out of range", max_ctx);
  if (n_seqs * max_ctx >> 32)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "attention_tree: %zu sequences of %zu rows (together less than 2^32)", n_seqs,
                         max_ctx);
  if (ldq < n_heads * head_dim || ldkv < n_kv_heads * head_dim)
    return wh::set_error(WH_ERR_INVALID_SHAPE, "attention_tree: row strides %zu, %zu below the rows' %zu, %zu elements",
                         ldq, ldkv, n_heads * head_dim, n_kv_heads * head_dim);
  if (n_seqs == 0 || n_tree == 0) return WH_OK;
  if (!q || !k || !v || !parents || !ctx_len || !k_cache || !v_cache || !inv_freq || !out || !workspace)
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "attention_tree: null pointer");
  if (!wh::aligned(k_cache, 16) || !wh::aligned(v_cache, 16) || !wh::aligned(workspace, 16))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "attention_tree: caches and workspace must be 16-byte aligned");
  if (!wh::aligned(q, 4) || !wh::aligned(k, 4) || !wh::aligned(v, 4) || !wh::aligned(parents, 4) ||
      !wh::aligned(ctx_len, 4) || !wh::aligned(inv_freq, 4) || !wh::aligned(out, 4))
    return wh::set_error(WH_ERR_INVALID_ARGUMENT, "attention_tree: arrays must be 4-byte aligned");
  const size_t need = wh::tree_attention_workspace_bytes(n_seqs, n_tree, n_heads, n_kv_heads, head_dim, max_ctx);
  if (workspace_bytes < need)
    return wh::set_error(WH_ERR_BUFFER_TOO_SMALL, "attention_tree: workspace too small: needed %zu bytes, available %zu",
                         need, workspace_bytes);
  const wh::TreeAttnArgs a{q,       k,       v,       ldq,       ldkv,     parents,    ctx_len,  n_seqs, n_tree,
                           k_cache, v_cache, max_ctx, n_heads, n_kv_heads, head_dim, inv_freq, out};
  return wh::launch_tree_attention(a, workspace, reinterpret_cast<hipStream_t>(stream));
}
