// paged_dev.h — device helpers that the paged-cache kernels (paged.hip,
// tree_attn.hip) share. Not public ABI.
#pragma once
#include "dev_common.h"

namespace wl {
namespace paged {

WL_DEV void set_status(uint32_t* status, uint32_t bits) {
    if (status && bits) __hip_atomic_fetch_or(status, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

WL_DEV uint32_t pack_bf16(float a, float b) {  // a in the low half
    bf16x2 r;
    r[0] = (__bf16)a;  // round to nearest even
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
}

}  // namespace paged
}  // namespace wl
