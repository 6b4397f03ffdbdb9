// paged.hip — the page map of a step (wl_paged_map), the write of its latent
// cache rows (wl_paged_write) and their reading back (wl_paged_read).
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "paged.h"
#include "paged_dev.h"

namespace wl {
namespace paged {
namespace {

// ---- the page map ---------------------------------------------------------
// One launch. With n = len, a = add, h = have of a request and w = ceil((n +
// a) / ps) the pages it needs, the step is three exclusive sums over the
// requests: of a (the tokens' ranges), of max(0, h - w) (where a request's
// surplus pages go on the stack) and of max(0, w - h) (which pages from the
// top it takes: the k-th of them all is stack[F - 1 - k], F = n_free + the
// surplus). Every work-group computes all three for itself from the lengths
// (12 bytes a request), so nothing is handed from one to another and the
// outputs are written in the same launch: the k-th page, when it is one that
// this step pushes, is looked up in the table it comes from, not on the stack.
// In a call with trees a wave takes a request, lane i its node i; otherwise a
// thread takes a token, or four, and finds its request by bisection.
// Bound by the launch and by latencies one after the other (lengths, the sums over
// the requests, page, slot), not by bytes: 8 requests of up to 8 nodes 3.8 us (an empty
// kernel takes 1.4); 256 of up to 64 nodes, 5083 in all, 5.8 us; 1000 prompts, 661k
// tokens, 5.3 MB out, 11 us (14.8 with one token a thread), of which the search over all
// requests for every four tokens is most.
struct Sums {
    uint64_t tok;
    uint32_t back, take;
};
WL_DEV Sums operator+(const Sums& a, const Sums& b) { return Sums{a.tok + b.tok, a.back + b.back, a.take + b.take}; }
WL_DEV Sums shfl_up(const Sums& s, uint32_t o) {
    Sums r;
    r.tok = (uint64_t)__shfl_up((unsigned long long)s.tok, o, 64);
    r.back = __shfl_up(s.back, o, 64);
    r.take = __shfl_up(s.take, o, 64);
    return r;
}

typedef __attribute__((ext_vector_type(4))) int32_t i32x4;
constexpr uint32_t kMapGrid = 512;  // work-groups at the most
// A thread takes four consecutive tokens, and searches once for their request, where
// a step holds many more of them than requests and one each would be more threads
// than half of the chip's places; otherwise one, so that lookups do not queue up in a
// thread. Token each / four each: 200 requests with 126k tokens 5.6 / 7.5 us, 1000
// with 165k 8.3 / 11.5, 327k 12.2 / 11.2, 661k 14.8 / 11.0; 256 with 1345 5.4 / 8.3.
__host__ __device__ inline bool runs_of_4(const wl_page_map& m) {
    return m.max_tokens >= 64u * m.n_req && m.max_tokens > (1u << 18);
}

template <uint32_t THREADS, uint32_t RPT>
__global__ __launch_bounds__(THREADS) void page_map_kernel(wl_page_map m) {
    constexpr uint32_t CAP = THREADS * RPT, NW = THREADS / 64;
    __shared__ uint32_t cu[CAP + 1], back[CAP + 1], take[CAP + 1], need[CAP], have[CAP], len[CAP];
    __shared__ Sums wsum[NW];
    __shared__ uint32_t err;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6, R = m.n_req;
    const uint32_t psh = 31u - (uint32_t)__clz((int)m.page_size), pmask = m.page_size - 1u;
    const bool trees = m.d_parent || m.d_mask;
    const int32_t nf = *m.d_n_free;
    if (tid == 0) err = 0;
    __syncthreads();
    // thread tid's requests are [RPT tid, RPT tid + RPT)
    Sums own[RPT], mine{0, 0, 0};
    uint32_t bad = 0;
#pragma unroll
    for (uint32_t i = 0; i < RPT; i++) {
        const uint32_t r = tid * RPT + i;
        own[i] = Sums{0, 0, 0};
        if (r < R) {
            const int32_t n = m.d_len[r], a = m.d_add[r], h = m.d_have[r];
            const uint64_t w = n < 0 || a < 0 ? 0 : ((uint64_t)n + (uint64_t)a + pmask) >> psh;
            const uint64_t filled = n < 0 ? 0 : ((uint64_t)n + pmask) >> psh;
            // an ended request (n = 0) may hold any number of pages
            if (n < 0 || a < 0 || h < 0 || (uint32_t)h > m.max_pages || w > m.max_pages || (uint64_t)(uint32_t)h < filled) {
                bad |= WL_PAGED_E_LEN;
            } else {
                if (trees && a > WL_TREE_MAX_NODES) bad |= WL_PAGED_E_TREE;
                own[i].tok = (uint64_t)a;
                own[i].back = (uint32_t)h > (uint32_t)w ? (uint32_t)h - (uint32_t)w : 0u;
                own[i].take = (uint32_t)w > (uint32_t)h ? (uint32_t)w - (uint32_t)h : 0u;
                need[r] = (uint32_t)w;
                have[r] = (uint32_t)h;
                len[r] = (uint32_t)n;
            }
        }
        mine = mine + own[i];
    }
    if (bad) atomicOr(&err, bad);
    Sums inc = mine;
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const Sums v = shfl_up(inc, o);
        if (lane >= o) inc = inc + v;
    }
    if (lane == 63) wsum[wv] = inc;
    __syncthreads();
    Sums at{inc.tok - mine.tok, inc.back - mine.back, inc.take - mine.take}, all{0, 0, 0};
#pragma unroll
    for (uint32_t w = 0; w < NW; w++) {
        if (w < wv) at = at + wsum[w];
        all = all + wsum[w];
    }
#pragma unroll
    for (uint32_t i = 0; i < RPT; i++) {
        const uint32_t r = tid * RPT + i;
        cu[r] = (uint32_t)at.tok;  // wraps only in a refused step
        back[r] = at.back;
        take[r] = at.take;
        at = at + own[i];
    }
    if (tid == THREADS - 1) {
        cu[CAP] = (uint32_t)at.tok;
        back[CAP] = at.back;
        take[CAP] = at.take;
    }
    uint32_t refuse = err;  // set before the barrier above
    if (all.tok > m.max_tokens) refuse |= WL_PAGED_E_LEN;
    if (nf < 0 || (uint32_t)nf > m.n_pages || (uint64_t)(uint32_t)nf + all.back > m.n_pages) refuse |= WL_PAGED_E_PAGE;
    else if (all.take > (uint32_t)nf + all.back) refuse |= WL_PAGED_E_SPACE;
    __syncthreads();
    const uint32_t gt = blockIdx.x * THREADS + tid, gn = gridDim.x * THREADS;
    if (refuse) {
        for (uint32_t r = gt; r < R; r += gn) m.d_have_out[r] = m.d_have[r];
        for (uint32_t r = gt; r <= R; r += gn) m.d_cu[r] = 0;
        for (uint32_t t = gt; t < m.max_tokens; t += gn) m.d_slot[t] = -1;
        if (gt == 0) {
            *m.d_n_free_out = nf;
            set_status(m.d_status, refuse);
        }
        return;
    }
    const uint32_t F = (uint32_t)nf + all.back, total = (uint32_t)all.tok;
    for (uint32_t r = gt; r < R; r += gn) m.d_have_out[r] = (int32_t)need[r];
    for (uint32_t r = gt; r <= R; r += gn) m.d_cu[r] = (int32_t)cu[r];
    if (gt == 0) *m.d_n_free_out = (int32_t)(F - all.take);
    for (uint32_t t = total + gt; t < m.max_tokens; t += gn) {  // behind the step's tokens: none
        m.d_slot[t] = -1;
        if (m.d_pos) m.d_pos[t] = 0;
    }
    // the last r with base[r] <= x: the owner of element x (empty ranges before it share its base)
    auto owner = [&](const uint32_t* base, uint32_t x) {
        uint32_t lo = 0, hi = R;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (base[mid] <= x) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    auto pushed = [&](uint32_t j) {  // the j-th page that this step pushes
        const uint32_t r = owner(back, j);
        return m.d_table[(size_t)r * m.max_pages + need[r] + (j - back[r])];
    };
    uint32_t flaw = 0;
    auto in_cache = [&](int32_t page) { return page >= 0 && (uint32_t)page < m.n_pages; };
    for (uint32_t j = gt; j < all.back; j += gn) {  // what is no page is told of here, and given back all the same
        const int32_t page = pushed(j);
        if (!in_cache(page)) flaw |= WL_PAGED_E_PAGE;
        m.d_free[(uint32_t)nf + j] = page;
    }
    // the slot of token i of request r; the first token of a new page writes the table's entry
    auto place = [&](uint32_t r, uint32_t i) {
        const uint32_t row = len[r] + i, k = row >> psh;
        int32_t page;
        if (k < have[r]) {
            page = m.d_table[(size_t)r * m.max_pages + k];
        } else {
            const uint32_t s = F - 1u - (take[r] + (k - have[r]));
            page = s >= (uint32_t)nf ? pushed(s - (uint32_t)nf) : m.d_free[s];
            if ((row & pmask) == 0) m.d_table[(size_t)r * m.max_pages + k] = page;
        }
        const bool ok = in_cache(page);
        if (!ok) flaw |= WL_PAGED_E_PAGE;
        return ok ? (int32_t)(((uint32_t)page << psh) + (row & pmask)) : -1;
    };
    if (trees) {
        for (uint32_t r = blockIdx.x * NW + wv; r < R; r += gridDim.x * NW) {
            const uint32_t t0 = cu[r], a = cu[r + 1] - t0, i = lane;
            const uint32_t t = t0 + (i < a ? i : 0u);
            int32_t up = (int32_t)i - 1;
            if (m.d_parent && i < a) {
                up = m.d_parent[t];
                if (up < -1 || up >= (int32_t)i) {
                    flaw |= WL_PAGED_E_TREE;
                    up = -1;
                }
            }
            // pointer doubling: after step s the mask covers 2^s generations
            uint64_t bits = 1ull << i;
            uint32_t depth = up >= 0 ? 1u : 0u;
#pragma unroll
            for (int s = 0; s < 6; s++) {
                const int from = up >= 0 ? up : 0;
                const uint64_t b = (uint64_t)__shfl((unsigned long long)bits, from, 64);
                const uint32_t d = __shfl(depth, from, 64);
                const int32_t u = __shfl(up, from, 64);
                if (up >= 0) {
                    bits |= b;
                    depth += d;
                    up = u;
                }
            }
            if (i < a) {
                m.d_slot[t] = place(r, i);
                if (m.d_mask) m.d_mask[t] = bits;
                if (m.d_pos) m.d_pos[t] = (int32_t)(len[r] + depth);
            }
        }
    } else if (runs_of_4(m)) {
        const bool wide = (((uintptr_t)m.d_slot | (uintptr_t)m.d_pos) & 15u) == 0;
        for (uint32_t t = 4u * gt; t < total; t += 4u * gn) {
            uint32_t r = owner(cu, t);
            int32_t slot[4], pos[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                if (t + k >= total) break;
                uint32_t i = t + k - cu[r];
                bool same = k > 0;
                while (t + k >= cu[r + 1]) {  // on to its request: cu[R] is behind all of them
                    i = t + k - cu[++r];
                    same = false;
                }
                if (same && ((len[r] + i) & pmask)) slot[k] = slot[k ? k - 1 : 0] + (slot[k ? k - 1 : 0] >= 0 ? 1 : 0);
                else slot[k] = place(r, i);
                pos[k] = (int32_t)(len[r] + i);
            }
            if (wide && t + 4u <= total) {
                *(i32x4*)(m.d_slot + t) = i32x4{slot[0], slot[1], slot[2], slot[3]};
                if (m.d_pos) *(i32x4*)(m.d_pos + t) = i32x4{pos[0], pos[1], pos[2], pos[3]};
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) {
                    if (t + k >= total) break;
                    m.d_slot[t + k] = slot[k];
                    if (m.d_pos) m.d_pos[t + k] = pos[k];
                }
            }
        }
    } else {
        for (uint32_t t = gt; t < total; t += gn) {
            const uint32_t r = owner(cu, t), i = t - cu[r];
            m.d_slot[t] = place(r, i);
            if (m.d_pos) m.d_pos[t] = (int32_t)(len[r] + i);
        }
    }
    set_status(m.d_status, flaw);
}

// ---- the write of cache rows ------------------------------------------------
// A wave holds a token's row in registers: lane l the values [8 l, 8 l + 8) of
// the compressed part (one pass: square sum over the wave, scale, store) and,
// in lanes below RP / 8, 4 pairs of the rotary part. Lane i < RP / 2 computes
// the angle of pair i: pos * theta^(-2 i / RP) in 64 bits, less its whole
// turns, then sine and cosine of the rest in f32 with the rest's own rounding
// added to first order; the other lanes take the pairs' values by permutes.
// Bound by the bytes: 16384 bf16 tokens with 64 heads' queries, 306 MB read and
// written in 61.4 us, 4.98 TB/s (a large copy: 5.05). 333 tokens 5.3 us, one token
// 3.7 us: a kernel's 1.4 and two trips to memory (3.9 with the row called for only
// when its slot had come).
struct RowWrite {
    wl_row_write w;
    double inv[kMaxRope / 2];  // theta^(-2 i / qk_rope)
    uint32_t wpt;              // waves per token
};

WL_DEV void sincos_of(double ang, float& s, float& c) {
    const double turns = rint(ang * 0.15915494309189533577);        // 1 / (2 pi)
    double x = fma(-turns, 6.283185307179586232, ang);              // 2 pi, its leading 53 bits
    x = fma(-turns, 2.4492935982947064e-16, x);                     // and the rest
    const float h = (float)x, d = (float)(x - (double)h);
    float s0, c0;
    sincosf(h, &s0, &c0);
    s = s0 + d * c0;
    c = c0 - d * s0;
}

template <bool BF>
WL_DEV void load8(const void* p, size_t i, float* v) {
    if (BF) {
        const u32x4 x = gld16((const uint16_t*)p + i);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[2 * k] = __uint_as_float(x[k] << 16);
            v[2 * k + 1] = __uint_as_float(x[k] & 0xFFFF0000u);
        }
    } else {
        const u32x4 a = gld16((const float*)p + i), b = gld16((const float*)p + i + 4);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[k] = __uint_as_float(a[k]);
            v[4 + k] = __uint_as_float(b[k]);
        }
    }
}
template <int N>
WL_DEV void store_n(void* p, size_t i, const float* v, bool bf) {
    if (bf) {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
            const u32x2 x = {pack_bf16(v[k], v[k + 1]), pack_bf16(v[k + 2], v[k + 3])};
            gst((u32x2*)((uint16_t*)p + i + k), x);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k += 4) gst((f32x4*)((float*)p + i + k), f32x4{v[k], v[k + 1], v[k + 2], v[k + 3]});
    }
}

// The compressed part of a row of a 4-bit cache, a lane's 8 values v with weights g:
// everything in 64 bits, so that a value is on the side of a border between two 4-bit
// ones that its exact value is on (in 32 bits about one in 2^20 is not, and a step is a
// third of the value). Four lanes hold a block. Its 7 64-bit comparisons a value are hidden
// behind the bytes: 13725 tokens of 64 heads, bf16, 246 MB, 49 us, the rate of 16-bit rows.
WL_DEV void store_mx(uint8_t* row, uint32_t lane, uint32_t L, const float* v, const float* g, float eps) {
    double c[8], ss = 0.0;
#pragma unroll
    for (int k = 0; k < 8; k++) ss += (double)v[k] * (double)v[k];
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    const double rs = 1.0 / sqrt(ss / (double)L + (double)eps);
    double most = 0.0;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        c[k] = (double)v[k] * rs * (double)g[k];
        bad |= !(fabs(c[k]) < INFINITY);
        most = fmax(most, fabs(c[k]));
    }
    uint32_t nf = bad ? 1u : 0u;
    for (int o = 1; o < 4; o <<= 1) {
        most = fmax(most, __shfl_xor(most, o, 64));
        nf |= __shfl_xor(nf, o, 64);
    }
    // the least e with most <= 6 2^e: 6 is 3/2 of 4
    const uint64_t bits = (uint64_t)__double_as_longlong(most);
    int32_t e = (int32_t)(bits >> 52) - 1023 - 2 + ((bits & 0xFFFFFFFFFFFFFull) > 0x8000000000000ull ? 1 : 0);
    e = e < (int32_t)kMxLo - 127 ? (int32_t)kMxLo - 127 : e > (int32_t)kMxHi - 127 ? (int32_t)kMxHi - 127 : e;
    const double inv = __longlong_as_double((int64_t)(1023 - e) << 52);
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const double a = fabs(c[k]) * inv;
        const uint32_t code = (a > 0.25 ? 1u : 0u) + (a >= 0.75 ? 1u : 0u) + (a > 1.25 ? 1u : 0u) + (a >= 1.75 ? 1u : 0u) +
                              (a > 2.5 ? 1u : 0u) + (a >= 3.5 ? 1u : 0u) + (a > 5.0 ? 1u : 0u);
        word |= (code | (code && c[k] < 0.0 ? 8u : 0u)) << (4 * k);
    }
    if (8u * lane < L) gst((uint32_t*)row + lane, word);
    // lane j < 4 has the scales of blocks j, 4 + j, 8 + j and 12 + j, each from its block's first lane
    const uint32_t mine = 8u * lane < L ? (nf ? 255u : (uint32_t)(e + 127)) : 0u;
    uint32_t scales = 0;
#pragma unroll
    for (uint32_t s = 0; s < 4; s++) scales |= __shfl(mine, (int)(16u * s + 4u * (lane & 3u)), 64) << (8u * s);
    if (lane < 4) gst((uint32_t*)(row + L / 2) + lane, scales);
}

template <bool BF, bool MX>
__global__ __launch_bounds__(256) void row_write_kernel(RowWrite a) {
    const wl_row_write& w = a.w;
    const uint32_t lane = threadIdx.x & 63u, wave = blockIdx.x * 4u + (threadIdx.x >> 6);
    const uint32_t t = wave / a.wpt, part = wave % a.wpt;
    if (t >= w.n_tokens) return;
    const uint32_t L = w.cache.kv_lora_rank, RP = w.cache.qk_rope, HP = RP / 2;
    const bool cbf = w.cache.dtype == WL_TYPE_BF16;
    // everything the wave needs first is called for before anything is waited for
    const int32_t pos = w.d_pos[t], slot = part == 0 ? w.d_slot[t] : -1, src = part == 0 && w.d_src ? w.d_src[t] : (int32_t)t;
    const uint32_t cph = RP / 8, vpw = 64 / cph, c = lane % cph, vl = lane / cph;
    const uint32_t i = 8 * lane;
    const bool src_ok = !w.d_src || (src >= 0 && (uint32_t)src < w.n_kv);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, r[8], g[8], qv[8];
    if (part == 0 && src_ok) {
        const size_t in = (size_t)src * w.kv_stride;
        if (i < L) {
            load8<BF>(w.d_kv, in + i, v);
            load8<true>(w.d_norm_w, i, g);
        }
        if (lane < cph) load8<BF>(w.d_kv, in + L + i, r);
    }
    auto load_q = [&](uint32_t h0) {
        if (vl < vpw && h0 + vl < w.n_heads) load8<BF>(w.d_q_rope, (size_t)t * w.q_stride + (size_t)(h0 + vl) * RP + 8 * c, qv);
    };
    load_q(part * vpw);
    if (pos < 0) {
        if (lane == 0 && part == 0) set_status(w.d_status, WL_PAGED_E_LEN);
        return;
    }
    float sn = 0.f, cs = 0.f;
    if (lane < HP) sincos_of((double)pos * a.inv[lane], sn, cs);
    // this lane's 4 pairs: chunk c of the RP / 8 chunks of a rotary vector, of vector vl of the wave's vpw
    float s4[4], c4[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        s4[k] = __shfl(sn, 4 * c + k, 64);
        c4[k] = __shfl(cs, 4 * c + k, 64);
    }
    auto turn = [&](const float* v, float* lo, float* hi) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            lo[k] = v[2 * k] * c4[k] - v[2 * k + 1] * s4[k];
            hi[k] = v[2 * k + 1] * c4[k] + v[2 * k] * s4[k];
        }
    };
    if (part == 0) {
        const uint32_t rows = w.cache.n_pages * w.cache.page_size;
        const bool bad = slot < -1 || (slot >= 0 && ((uint32_t)slot >= rows || !src_ok));
        if (bad && lane == 0) set_status(w.d_status, WL_PAGED_E_SLOT);
        if (MX && !bad && slot >= 0) {
            uint8_t* row = (uint8_t*)w.cache.d_rows + (size_t)slot * w.cache.row_stride;
            if (i >= L) {
#pragma unroll
                for (int k = 0; k < 8; k++) g[k] = 0.f;
            }
            store_mx(row, lane, L, v, g, w.eps);
            if (lane < cph) {
                float lo[4], hi[4];
                turn(r, lo, hi);
                store_n<4>(row + L / 2 + kMxScales, 4 * c, lo, true);
                store_n<4>(row + L / 2 + kMxScales, HP + 4 * c, hi, true);
            }
        }
        if (!MX && !bad && slot >= 0) {
            const size_t out = (size_t)slot * w.cache.row_stride;
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) ss += v[k] * v[k];
            for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
            const float rs = 1.0f / sqrtf(ss / (float)L + w.eps);
            if (i < L) {
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = g[k] * (v[k] * rs);
                store_n<8>(w.cache.d_rows, out + i, v, cbf);
            }
            if (lane < cph) {
                float lo[4], hi[4];
                turn(r, lo, hi);
                store_n<4>(w.cache.d_rows, out + L + 4 * c, lo, cbf);
                store_n<4>(w.cache.d_rows, out + L + HP + 4 * c, hi, cbf);
            }
        }
    }
    // a wave's heads come vpw at a time; a vector is read whole before any of
    // it is written (its lanes are one wave's), so the output may be the input
    for (uint32_t h0 = part * vpw; h0 < w.n_heads; h0 += a.wpt * vpw) {
        const uint32_t h = h0 + vl;
        const bool ok = vl < vpw && h < w.n_heads;
        float lo[4], hi[4];
        if (h0 != part * vpw) load_q(h0);
        __builtin_amdgcn_wave_barrier();
        if (ok) {
            turn(qv, lo, hi);
            const size_t out = (size_t)t * w.q_out_stride + (size_t)h * RP + 4 * c;
            store_n<4>(w.d_q_rope_out, out, lo, BF);
            store_n<4>(w.d_q_rope_out, out + HP, hi, BF);
        }
    }
}

// ---- rows as values -----------------------------------------------------------
// A thread has 8 values of a row, so a row's chunks, the rotary ones among them, lie in
// a row over the threads; a request's are dealt out to the work-groups of its row of the
// grid. Where a request may be much longer than the others (REST), these take `most` chunks
// of it, and what is behind them is dealt out to the work-groups of the grid's first
// rows, 256 chunks at a time, beginning elsewhere for each request: these look through the
// requests for long ones. Bound by the launch (one row 2.2 us in a row of calls), then by
// the bytes: 13725 rows of 4 bits to bf16, 21 MB, 6.8 us; of 16 bits to bf16, 32 MB, 6.4;
// of 32 bits to 32 bits, 63 MB, 11.9; 32768 rows of these 12.4, 13.1 and 24.2 us (6.2 TB/s).
struct RowRead {
    wl_row_read r;
    uint32_t psh;    // log2 page_size
    uint32_t most;   // chunks of a request that its own work-groups read (REST)
    uint32_t rest;   // work-groups for the others,
    uint32_t first;  // and rows of the grid
};

template <int CT, bool OBF, bool REST>
__global__ __launch_bounds__(256) void row_read_kernel(RowRead a) {
    constexpr bool MX = CT == WL_TYPE_MXFP4;
    const wl_row_read& p = a.r;
    const uint32_t psh = a.psh, tid = threadIdx.x, L = p.cache.kv_lora_rank, RP = p.cache.qk_rope, cl = L / 8u, per = cl + RP / 8u;
    // whether request r has rows that can be, in c0, c1 and first
    auto sound = [&](int32_t c0, int32_t c1, int32_t first) {
        return c0 >= 0 && c1 >= c0 && (uint32_t)c1 <= p.n_rows && first >= 0 &&
               (uint64_t)(uint32_t)first + (uint32_t)(c1 - c0) <= ((uint64_t)p.max_pages << psh);
    };
    // chunk i of request r, whose rows begin with row c0 and token `first`
    auto chunk = [&](uint32_t r, uint32_t c0, uint32_t first, uint32_t i) {
        const uint32_t j = i / per, k = i - j * per, key = first + j;
        const int32_t page = p.d_table[(size_t)r * p.max_pages + (key >> psh)];
        float v[8];
        if (page < 0 || (uint32_t)page >= p.cache.n_pages) {
            if (k == 0) set_status(p.d_status, WL_PAGED_E_PAGE);
#pragma unroll
            for (int m = 0; m < 8; m++) v[m] = __builtin_nanf("");
        } else {
            const size_t at = (((size_t)(uint32_t)page << psh) + (key & (p.cache.page_size - 1u))) * p.cache.row_stride;
            if (MX) {
                const uint8_t* row = (const uint8_t*)p.cache.d_rows + at;
                if (k < cl) {
                    const uint32_t s = gld1(row + L / 2 + mx_scale_at(k / 4u));
                    const u32x4 x = __builtin_bit_cast(u32x4, fp4x8_bf16(gld((const uint32_t*)row + k), e8m0f(s)));
#pragma unroll
                    for (int m = 0; m < 4; m++) {
                        v[2 * m] = s > kMxHi ? __builtin_nanf("") : __uint_as_float(x[m] << 16);
                        v[2 * m + 1] = s > kMxHi ? __builtin_nanf("") : __uint_as_float(x[m] & 0xFFFF0000u);
                    }
                } else {
                    load8<true>(row + L / 2 + kMxScales, 8u * (k - cl), v);
                }
            } else {
                load8<CT == WL_TYPE_BF16>(p.cache.d_rows, at + 8u * k, v);
            }
        }
        store_n<8>(p.d_out, (size_t)(c0 + j) * p.out_stride + 8u * k, v, OBF);
    };
    if (!REST || blockIdx.y >= a.first) {
        const uint32_t r = blockIdx.y - (REST ? a.first : 0u);
        const int32_t c0 = p.d_cu[r], c1 = p.d_cu[r + 1], first = p.d_first ? p.d_first[r] : 0;
        if (c0 == c1) return;
        if (!sound(c0, c1, first)) {
            if (blockIdx.x == 0 && tid == 0) set_status(p.d_status, WL_PAGED_E_LEN);
            return;
        }
        const uint32_t all = (uint32_t)(c1 - c0) * per, n = !REST || all < a.most ? all : a.most;  // n_rows <= 2^24, per <= 72
        for (uint32_t i = blockIdx.x * 256u + tid; i < n; i += gridDim.x * 256u) chunk(r, (uint32_t)c0, (uint32_t)first, i);
        return;
    }
    if constexpr (REST) {
        constexpr uint32_t EACH = WL_PAGED_MAX_REQ / 256u;  // requests of a thread
        __shared__ uint16_t list[WL_PAGED_MAX_REQ];         // long requests with chunks for this work-group
        __shared__ uint32_t count;
        const uint32_t h = blockIdx.y * gridDim.x + blockIdx.x;
        // which 256 of the rest's chunks are the work-group's first of request r
        auto place = [&](uint32_t r) {
            const uint32_t from = (r * 0x9E3779B1u >> 16) % a.rest;
            return h >= from ? h - from : h + a.rest - from;
        };
        auto blocks = [&](uint32_t all) { return (all - a.most + 255u) / 256u; };
        if (h >= a.rest) return;
        if (tid == 0) count = 0;
        int32_t c0[EACH], c1[EACH];
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++) {
            const uint32_t r = 256u * k + tid;
            c0[k] = c1[k] = 0;
            if (256u * k < p.n_req && r < p.n_req) {
                c0[k] = p.d_cu[r];
                c1[k] = p.d_cu[r + 1];
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++) {
            if (c1[k] <= c0[k] || c0[k] < 0 || (uint32_t)c1[k] > p.n_rows) continue;
            const uint32_t r = 256u * k + tid, all = (uint32_t)(c1[k] - c0[k]) * per;
            if (all > a.most && place(r) < blocks(all) && sound(c0[k], c1[k], p.d_first ? p.d_first[r] : 0))
                list[atomicAdd(&count, 1u)] = (uint16_t)r;  // (their order changes no result)
        }
        __syncthreads();
        for (uint32_t l = 0; l < count; l++) {
            const uint32_t r = uni(list[l]), c = (uint32_t)p.d_cu[r], all = ((uint32_t)p.d_cu[r + 1] - c) * per;
            const uint32_t first = p.d_first ? (uint32_t)p.d_first[r] : 0u;
            for (uint32_t b = place(r); b < blocks(all); b += a.rest) {
                const uint32_t i = a.most + 256u * b + tid;
                if (i < all) chunk(r, c, first, i);
            }
        }
    }
}

}  // namespace

int launch_read(const wl_row_read& r, void* stream) {
    const uint32_t per = (r.cache.kv_lora_rank + r.cache.qk_rope) / 8u;
    RowRead a{};
    a.r = r;
    a.psh = 31u - (uint32_t)__builtin_clz(r.cache.page_size);
    // 4096 work-groups in all, as many for each request. One request alone may have all rows:
    // where that would be more than 24 rounds of its work-groups (some 0.7 us each), they take
    // twice those of an average request and four, and up to 512 others what is behind them. One
    // request with 65536 rows among 512, 4 bits: 2156 us without them and 47, 16 bits 1477 and 35.
    // Requests of the same length pay up to 4 % or 0.4 us: 64 x 1000 rows of 4 bits 20.5 us
    // and 20.7, 4096 x 16 20.4 and 21.2 (with 2048 others 21.6 and 23.7), 4096 x 1 4.7 and 5.1.
    const uint32_t need = (uint32_t)(((uint64_t)r.n_rows * per + 255u) / 256u), own = r.n_req >= 4096u ? 1u : 4096u / r.n_req;
    const uint32_t x = need < own ? need : own, rounds = 2u * ((need + 4095u) / 4096u) + 4u;
    a.most = x * rounds * 256u;  // below 2^32: at most 4096 x 2308 x 256
    if (x * (rounds > 24u ? rounds : 24u) < need) a.rest = need / 8u < 512u ? need / 8u : 512u;
    a.first = (a.rest + x - 1u) / x;
    const dim3 grid(x, a.first + r.n_req);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto ct) {
        constexpr int CT = decltype(ct)::value;
        auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a); };
        if (r.dtype == WL_TYPE_BF16) a.rest ? run(row_read_kernel<CT, true, true>) : run(row_read_kernel<CT, true, false>);
        else a.rest ? run(row_read_kernel<CT, false, true>) : run(row_read_kernel<CT, false, false>);
        return (int)hipGetLastError();
    };
    return r.cache.dtype == WL_TYPE_MXFP4  ? go(std::integral_constant<int, WL_TYPE_MXFP4>{})
           : r.cache.dtype == WL_TYPE_BF16 ? go(std::integral_constant<int, WL_TYPE_BF16>{})
                                           : go(std::integral_constant<int, WL_TYPE_F32>{});
}

int launch_map(const wl_page_map& m, void* stream) {
    const bool trees = m.d_parent || m.d_mask;
    // a wave per request or a thread per token, and one for every page that may be
    // given back (256 requests of which some end with 16176 pages: 4.7 us, 48 in one
    // work-group), but no more work-groups than the chip has places for
    const uint32_t R = m.n_req;
    auto grid = [&](uint32_t threads) {
        uint64_t work = trees ? (uint64_t)R * 64u : runs_of_4(m) ? (m.max_tokens + 3u) / 4u : m.max_tokens;
        if (work < m.n_pages) work = m.n_pages;
        const uint64_t g = (work + threads - 1) / threads;
        return dim3((uint32_t)(g < 1 ? 1 : g > 512 ? 512 : g));
    };
    // a request a thread; up to 256 in small work-groups (8 requests 3.8 us, 5.1 in
    // large ones; 200 of up to 64 tokens 5.4 and 6.5)
    hipStream_t st = (hipStream_t)stream;
    if (R <= 256) hipLaunchKernelGGL((page_map_kernel<256, 1>), grid(256), dim3(256), 0, st, m);
    else if (R <= 1024) hipLaunchKernelGGL((page_map_kernel<1024, 1>), grid(1024), dim3(1024), 0, st, m);
    else hipLaunchKernelGGL((page_map_kernel<1024, 4>), grid(1024), dim3(1024), 0, st, m);
    return (int)hipGetLastError();
}

int launch_write(const wl_row_write& w, void* stream) {
    RowWrite a{};
    a.w = w;
    for (uint32_t i = 0; i < w.cache.qk_rope / 2; i++)
        a.inv[i] = 1.0 / std::pow((double)w.rope_theta, (double)(2 * i) / (double)w.cache.qk_rope);
    // a wave for every round of the heads, four at the most: more loads in flight. With
    // one / four, 64 heads: 333 32-bit tokens 7.2 / 5.6 us, 1500 13.1 / 10.9, 8192
    // 65 / 59; bf16 800 8.0 / 6.0, 8192 33.4 / 33.6, 16384 61.4 / 61.5
    const uint32_t vpw = 64u / (w.cache.qk_rope / 8u), rounds = (w.n_heads + vpw - 1u) / vpw;
    a.wpt = rounds < 1 ? 1 : rounds > 4 ? 4 : rounds;
    const uint32_t wgs = (uint32_t)(((uint64_t)w.n_tokens * a.wpt + 3) / 4);
    hipStream_t st = (hipStream_t)stream;
    const bool mx = w.cache.dtype == WL_TYPE_MXFP4;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(wgs), dim3(256), 0, st, a); };
    if (w.dtype == WL_TYPE_BF16) mx ? go(row_write_kernel<true, true>) : go(row_write_kernel<true, false>);
    else mx ? go(row_write_kernel<false, true>) : go(row_write_kernel<false, false>);
    return (int)hipGetLastError();
}

}  // namespace paged
}  // namespace wl
