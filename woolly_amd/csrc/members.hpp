// members.hpp -- launchers of the operators that run several continuations of
// one prompt (rope.hip, shared_attention.hip, beam.hip, members_step.hip).
// Arguments have been checked by the C entry points; the launchers choose
// kernels and launch them.
#pragma once

#include <type_traits>

#include "wh_common.hpp"

namespace wh {

constexpr size_t kMaxMembers = WH_MAX_MEMBERS;
constexpr size_t kMaxBeams = WH_MAX_BEAMS;

struct RopeArgs {
  const float *q, *k, *v;      // [members * n_new] rows of ldq, ldkv elements
  size_t ldq, ldkv;
  const uint32_t* base_len;    // [members / n_per], null: 0
  const uint32_t* len;         // [members], null: n_new
  size_t n_members, n_per, n_new, n_heads, n_kv_heads, head_dim;
  float* q_out;                // null: not wanted
  size_t ldq_out;
  float* k_out;
  size_t ldk_out;
  void *k_cache, *v_cache;     // f16 [members][max_rows][n_kv_heads][head_dim]
  size_t max_rows;
};
// What of the rules the kernel takes can be checked without the call's other arguments.
int check_rope_rules(const char* fn, const wh_rope_rules& r, size_t head_dim);
int launch_rope(const wh_rope_rules& r, const RopeArgs& a, hipStream_t stream);

struct SharedAttnArgs {
  const float* q;              // [members] rows of ldq elements
  size_t ldq;
  const uint32_t* prefix_len;  // [groups]
  const uint32_t* own_len;     // [members]
  size_t n_groups, n_per;
  const void *k_prefix, *v_prefix;
  size_t max_prefix;
  const void *k_own, *v_own;
  size_t max_own, n_heads, n_kv_heads, head_dim;
  float* out;
};
bool shared_attention_shape_ok(size_t n_groups, size_t n_per, size_t n_heads, size_t n_kv_heads, size_t head_dim,
                               size_t max_prefix, size_t max_own);
size_t shared_attention_workspace_bytes(size_t n_groups, size_t n_per, size_t n_heads, size_t n_kv_heads,
                                        size_t head_dim, size_t max_prefix, size_t max_own);
int launch_shared_attention(const SharedAttnArgs& a, void* workspace, hipStream_t stream);

}  // namespace wh

namespace whd {

// Sum over the L lanes (32 or 64) that work together, in every one of them: swaps within rows of
// 16 lanes, then of rows and halves (as wave_join, tree.hpp).
template <int L>
__device__ __forceinline__ double lanes_sum_f64(double v) {
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
  if constexpr (L == 64) {
    const auto l32 = __builtin_amdgcn_permlane32_swap(lo(v), lo(v), false, false), h32 = __builtin_amdgcn_permlane32_swap(hi(v), hi(v), false, false);
    v = make(l32[0], h32[0]) + make(l32[1], h32[1]);
  }
  return v;
}

}  // namespace whd
