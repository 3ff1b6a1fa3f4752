// The attention passes behind rhip_attn_* (attn.hip), one translation unit
// each, and the choice of their kernel variants.
#pragma once

#include <algorithm>
#include <climits>
#include <type_traits>

#include "attn_device.hpp"

namespace rhip {

void attn_forward_run(const AttnArgs &a, int32_t dtype, bool vec, hipStream_t stream);
void attn_backward_run(const AttnArgs &a, int32_t dtype, bool vec, hipStream_t stream);
// The shape of a pass's launch: 32-row blocks per workgroup (W), tiles of 32 W
// rows, and the workgroups that share one tile of query rows (forward) or of
// keys (backward), whose partial sums are the workspace.
struct AttnPlan {
  int32_t waves; // W
  int64_t tiles;
  int32_t splits;
};
AttnPlan attn_forward_plan(const rhip_attn &d);
AttnPlan attn_queries_plan(const rhip_attn &d);
AttnPlan attn_keys_plan(const rhip_attn &d);

// 32-row blocks per workgroup of the kernels over query rows: as many as leave
// two workgroups for each CU, or one with two blocks (bf16: a workgroup's own
// tiles for each wave, W = 1, take twice the time of W = 2 at full width; fp32
// is bound by its products, and W = 1 spreads them best). 8 heads of 6000
// rows, 32 wide, dq: W = 4 110 us, W = 2 93; 8 of 3000, 128 wide, forward: W =
// 2 46 us, W = 1 76; fp32, 2 key heads of 9903 rows: W = 2 77 us, W = 1 53. Four
// times the rows before W = 4 in fp32: 8 heads of 8192 rows 281 us, 319; under a
// causal mask, 32 wide, 153 and 122, 64 wide, 12 heads, 556 and 555.
inline int32_t attn_waves(int64_t rows, int32_t kv_heads, int32_t dtype) {
  if (rows / 128 * kv_heads >= 512)
    return 4;
  return rows / 64 * kv_heads >= (dtype == RHIP_F32 ? 512 : 256) ? 2 : 1;
}

// f(T{}, head width of the variant, whether rows load in 16-byte chunks).
// Rows that do not (a width or a stride that is no multiple of 16 bytes, an
// unaligned view) load element by element into the widest tile of the type.
template <typename F> void with_attn(int32_t dtype, int32_t dim, bool vec, F &&f) {
  auto typed = [&](auto t) {
    if (!vec)
      f(t, std::integral_constant<int, kAttnMaxDim>{}, std::false_type{});
    else if (dim <= 32)
      f(t, std::integral_constant<int, 32>{}, std::true_type{});
    else if (dim <= 64)
      f(t, std::integral_constant<int, 64>{}, std::true_type{});
    else if (dim <= 96)
      f(t, std::integral_constant<int, 96>{}, std::true_type{});
    else
      f(t, std::integral_constant<int, 128>{}, std::true_type{});
  };
  if (dtype == RHIP_F32)
    typed(float{});
  else
    typed(__bf16{});
}

// Dynamic LDS, beside a kernel's own, that spreads 512 to 768 workgroups of
// four blocks over the chip. Workgroups are packed into a CU as long as their
// LDS fits, so these would fill some CUs and leave others idle; with an
// allocation that lets no more of them into a CU than each has to take, they
// spread. The count is the least that the rows can make: a tile of every 32 W.
// Rows of ragged sequences make some more, which follow the first. Heads of 64,
// four sequences of 2048: 8 heads (two a CU) forward 68 us packed, 55 spread, dq
// 75 and 62; 12 heads (three) 81 and 70, dq 86 and 87; 16 heads (four) 89 and
// 96, so no more than three. Twelve sequences of 650, 8 heads: 42 both ways,
// but the keys' kernel, which holds its workgroups longer, 43 and 56: it is
// left packed.
template <int W> unsigned spread_lds(const AttnArgs &a, int own) {
  constexpr int64_t kCus = 256;
  constexpr int kLdsBytes = 160 * 1024;
  const int64_t tiles = (a.n_q * (a.heads / a.kv_heads) + 32 * W - 1) / (32 * W);
  const int64_t each = (tiles * a.kv_heads + kCus - 1) / kCus;
  if (W < 4 || each < 2 || each > 3)
    return 0;
  const int fits = kLdsBytes / static_cast<int>(each + 1) + 1024; // each do, one more does not
  return fits > own ? static_cast<unsigned>(fits - own) : 0u;
}

// launch(args, workgroups) for a pass's tiles, in as many launches as their
// workgroups need (a great many short sequences on several heads).
template <typename F>
void attn_launches(const AttnArgs &args, const AttnPlan &plan, int threads, F &&launch) {
  AttnArgs a = args;
  if (plan.tiles > INT32_MAX)
    throw Error(RHIP_ERR_UNSUPPORTED, "too many tiles");
  a.tiles = static_cast<int32_t>(plan.tiles), a.splits = plan.splits;
  // attn_grid rounds up to whole rounds of the XCDs
  const int64_t units = max_groups(threads) / a.kv_heads - kXcds;
  if (units < a.splits)
    throw Error(RHIP_ERR_UNSUPPORTED, "too many heads");
  const int64_t step = units / a.splits;
  for (int64_t t = 0; t < plan.tiles; t += step) {
    a.tile0 = static_cast<int32_t>(t);
    a.launched = static_cast<int32_t>(std::min(step, plan.tiles - t));
    launch(a, static_cast<unsigned>(attn_grid(a.launched, a.kv_heads, a.splits)));
    RHIP_LAUNCH_CHECK();
  }
}

// f(W): 32-row blocks per workgroup, 4, 2 or 1.
template <typename F> void with_waves(int32_t waves, F &&f) {
  if (waves == 4)
    f(std::integral_constant<int, 4>{});
  else if (waves == 2)
    f(std::integral_constant<int, 2>{});
  else
    f(std::integral_constant<int, 1>{});
}

} // namespace rhip
