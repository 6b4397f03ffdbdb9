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
int launch_tree(const wl_tree_attn& a, void* stream);
size_t tree_scratch(const wl_tree_attn& a);

constexpr uint32_t kMaxRope = 64;

}  // namespace paged
}  // namespace wl
