// paged.h — launches of the paged-cache kernels (paged.hip, tree_attn.hip) for
// their host code (paged_host.cpp). Not public ABI.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "../../include/windlass_moe.h"

namespace wl {
namespace paged {

// Each returns the launch's hipError_t; the argument block has been checked.
int launch_map(const wl_page_map& m, void* stream);
int launch_write(const wl_row_write& w, void* stream);
int launch_tree(const wl_tree_attn& a, uint32_t window, uint32_t sinks, void* stream);  // window 0: none
int launch_tree_mx4(const wl_tree_attn& a, uint32_t window, uint32_t sinks, void* stream);  // 16-bit queries, 4-bit cache
size_t tree_scratch(const wl_tree_attn& a);
int launch_read(const wl_row_read& r, void* stream);
int launch_logprobs(const wl_logprobs& a, void* stream);
size_t logprobs_scratch(const wl_logprobs& a);

constexpr uint32_t kMaxRope = 64;
// A row of a 4-bit cache: kv_lora_rank / 2 bytes of values, kMxScales of their blocks'
// scales, the rotary part in 16 bits.
constexpr uint32_t kMxScales = 16;
// Where among them block b's stands: a lane of the scaled products has blocks g, 4 + g,
// 8 + g and 12 + g, whose scales are then one word.
constexpr uint32_t mx_scale_at(uint32_t b) { return 4u * (b % 4u) + b / 4u; }
constexpr uint32_t kMxLo = 2, kMxHi = 252;  // the scales that the write gives a block (above: a block that is NaN)

}  // namespace paged
}  // namespace wl
