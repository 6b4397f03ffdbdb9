// paged_dev.h — device helpers that the paged-cache kernels (paged.hip,
// tree_dev.h, tree_attn.hip, tree_mx4.hip, logprobs.hip) share. Not public ABI.
#pragma once
#include <type_traits>

#include "dev_common.h"
#include "paged.h"

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

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
// A block of 32 E2M1 values and its scale, on their way to bf16 (exact): 16-byte pieces
// j = 0 .. 3 go into LDS, piece (turn + j) % 4 of the block at dst. (The lanes of a wave
// write with different turns, so that they meet different banks.) A block that is NaN
// becomes zeros.
struct MxBlock {
    u32x4 x;
    float scale;
    uint32_t turn;
};
WL_DEV MxBlock mx_block(u32x4 x, uint32_t scale, uint32_t turn) {
    const bool t1 = turn & 1u, t2 = turn & 2u, nan = scale > kMxHi;
    const u32x4 y = t1 ? u32x4{x[1], x[2], x[3], x[0]} : x, z = t2 ? u32x4{y[2], y[3], y[0], y[1]} : y;
    return MxBlock{nan ? u32x4{0u, 0u, 0u, 0u} : z, __uint_as_float(nan ? 0u : scale << 23), turn};
}
WL_DEV void mx_put(const MxBlock& b, uint32_t j, uint8_t* dst) {
    *(u32x4*)(dst + 16u * ((b.turn + j) & 3u)) = __builtin_bit_cast(u32x4, fp4x8_bf16(b.x[j], b.scale));
}

// f(0), .., f(N - 1) with constants
template <int N, class F>
WL_DEV void static_for(F f) {
    if constexpr (N > 0) {
        static_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

}  // namespace paged
}  // namespace wl
