// tree_attn.hip — attention of trees of drafted tokens over a paged cache of
// latent rows (wl_paged_tree_attention).
#include <hip/hip_runtime.h>

#include "dev_common.h"
#include "paged.h"

namespace wl {
namespace paged {
namespace {

template <bool BF>
WL_DEV float ld1(const void* p, size_t i) {
    return BF ? bf2f(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}

// One wave per (request, node, head): lane l holds columns l, l + 64, ... of
// the query and of the output; one key after another, with the running
// maximum and sum of the softmax.
template <bool QBF, bool CBF>
__global__ __launch_bounds__(256) void tree_attn_kernel(wl_tree_attn a) {
    const uint32_t lane = threadIdx.x & 63u, wv = threadIdx.x >> 6;
    const uint32_t r = blockIdx.x, h = blockIdx.y * 4u + wv, node0 = blockIdx.z;
    if (h >= a.n_heads) return;
    const uint32_t L = a.cache.kv_lora_rank, W = L + a.cache.qk_rope, ps = a.cache.page_size;
    const int32_t t0 = a.d_cu[r], t1 = a.d_cu[r + 1], n = a.d_len[r];
    uint32_t bad = 0;
    if (t0 < 0 || t1 < t0 || (uint32_t)t1 > a.n_tokens) {
        if (a.d_status && lane == 0) atomicOr(a.d_status, WL_PAGED_E_LEN);
        return;
    }
    const uint32_t m = (uint32_t)(t1 - t0);
    if (m == 0) return;
    if (n < 0 || (uint64_t)n + m > (uint64_t)a.max_pages * ps) bad |= WL_PAGED_E_LEN;
    if (m > WL_TREE_MAX_NODES) bad |= WL_PAGED_E_TREE;
    const int32_t* table = a.d_table + (size_t)r * a.max_pages;
    const uint32_t K = bad ? 0u : (uint32_t)n + m;
    for (uint32_t k = lane; k * ps < K; k += 64)
        if (table[k] < 0 || (uint32_t)table[k] >= a.cache.n_pages) bad |= WL_PAGED_E_PAGE;
    for (int o = 32; o > 0; o >>= 1) bad |= __shfl_xor(bad, o, 64);
    if (bad && a.d_status && lane == 0) atomicOr(a.d_status, bad);
    for (uint32_t i = node0; i < m; i += gridDim.z) {
        const uint32_t t = (uint32_t)t0 + i;
        const uint64_t bits = a.d_mask ? a.d_mask[t] : (2ull << (i & 63u)) - 1ull;
        float q[9], acc[8], mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < 9; j++) {
            const uint32_t c = lane + 64 * j;
            q[j] = c < L ? ld1<QBF>(a.d_q_lat, t * a.q_lat_stride + (size_t)h * L + c)
                   : c < W ? ld1<QBF>(a.d_q_rope, t * a.q_rope_stride + (size_t)h * (W - L) + (c - L)) : 0.f;
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) acc[j] = 0.f;
        for (uint32_t k = 0; k < K && !bad; k++) {
            if (k >= (uint32_t)n && !((bits >> (k - (uint32_t)n)) & 1)) continue;
            const size_t row = ((size_t)(uint32_t)table[k / ps] * ps + k % ps) * a.cache.row_stride;
            float v[9], s = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < 9; j++) {
                const uint32_t c = lane + 64 * j;
                v[j] = c < W ? ld1<CBF>(a.cache.d_rows, row + c) : 0.f;
                s += q[j] * v[j];
            }
            for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            s *= a.scale;
            const float mn = s != s ? s : fmaxf(mx, s);
            const float al = mx == -INFINITY ? 0.f : expf(mx - mn), p = expf(s - mn);
            sum = sum * al + p;
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) acc[j] = acc[j] * al + p * v[j];
            mx = mn;
        }
        const float inv = bad ? __builtin_nanf("") : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            const uint32_t c = lane + 64 * j;
            if (c >= L) break;
            const size_t o = t * a.out_stride + (size_t)h * L + c;
            const float y = acc[j] * inv;
            if (QBF) ((uint16_t*)a.d_out)[o] = y != y ? 0x7FC0u : (uint16_t)f2bf(y);
            else ((float*)a.d_out)[o] = y;
        }
    }
}

}  // namespace

size_t tree_scratch(const wl_tree_attn&) { return 16; }

int launch_tree(const wl_tree_attn& a, void* stream) {
    const dim3 g(a.n_req, (a.n_heads + 3) / 4, 8);
    hipStream_t st = (hipStream_t)stream;
    if (a.dtype == WL_TYPE_BF16) hipLaunchKernelGGL((tree_attn_kernel<true, true>), g, dim3(256), 0, st, a);
    else if (a.cache.dtype == WL_TYPE_BF16) hipLaunchKernelGGL((tree_attn_kernel<false, true>), g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((tree_attn_kernel<false, false>), g, dim3(256), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace paged
}  // namespace wl
