// logprobs.hip — log probabilities of tokens under rows of logits, the rows'
// entropies and their most likely tokens (wl_token_logprobs).
#include <hip/hip_runtime.h>

#include "paged.h"
#include "paged_dev.h"

namespace wl {
namespace paged {
namespace {

// With M the largest logit of a row, S = sum exp(z - M) and U = sum exp(z - M) (z - M):
//   log p = z - M - log S, entropy = log S - U / S,
// and parts of a row with references m join as S = sum e^(m - M) s, U = sum e^(m - M)
// (u + (m - M) s). (Sums of exp times z itself would lose what z has over z - M.)
//
// First launch: a wave has a part of a row, one pass over it. A lane has 32 values at a
// time, their largest, and its own m, s and u, brought to a new m once for the 32. The
// n_top largest so far stand in the wave's lanes, in order: value as an ordered integer,
// id. What is at least the last of them (one comparison for each 8 values; few pass)
// goes in one by one: its place is the number of lanes before it, those behind take
// their neighbour's. The first 32 x 64 values' bound is the n_top-th of the lanes' largest:
// that many are at least as large. Second launch: a work-group a row joins its parts, a
// wave a token looks up its logit.
constexpr uint32_t kPer = 32;             // values a lane has at a time
constexpr uint32_t kPart = 64 * kPer;     // of a wave
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504088896340736f;

struct Logp {
    wl_logprobs a;
    uint32_t parts;   // per row
    float* sums;      // [n_rows][parts][4] m, s, u
    uint32_t* top;    // [n_rows][parts][n_top][2] ordered value, id
};

// Integers in the order of the values, NaN (any) the largest and -0 as +0; no value's is 0.
WL_DEV uint32_t ordered(float z) {
    const uint32_t u = __float_as_uint(z + 0.f);
    return z != z ? 0xFFFFFFFFu : (u >> 31) ? ~u : u | 0x80000000u;
}
WL_DEV float value_of(uint32_t o) {  // of 0: below any
    return o == 0xFFFFFFFFu ? __builtin_nanf("") : o == 0u ? -INFINITY : __uint_as_float(o >> 31 ? o & 0x7FFFFFFFu : ~o);
}
WL_DEV float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // a NaN, if one is

struct Sums {
    float m, s, u;
};
WL_DEV Sums to_reference(Sums x, float m) {  // m at least x.m, or NaN
    const float d = x.m - m, w = __builtin_amdgcn_exp2f(d * kLog2e);
    return Sums{m, w == 0.f ? 0.f : x.s * w, w == 0.f ? 0.f : w * fmaf(d, x.s, x.u)};
}
WL_DEV Sums join(Sums a, Sums b) {
    const float m = larger(a.m, b.m);
    const Sums x = to_reference(a, m), y = to_reference(b, m);
    return Sums{m, x.s + y.s, x.u + y.u};
}
WL_DEV Sums wave_join(Sums x) {
    for (int o = 32; o > 0; o >>= 1) x = join(x, Sums{__shfl_xor(x.m, o, 64), __shfl_xor(x.s, o, 64), __shfl_xor(x.u, o, 64)});
    return x;
}

// The largest of a wave's values so far: lane i the i-th.
struct Best {
    uint32_t key = 0, id = ~0u;
    float least = -INFINITY;  // what is below it is not among the n
    __device__ __forceinline__ bool before(uint32_t k, uint32_t i) const { return key > k || (key == k && id < i); }
    __device__ __forceinline__ void put(uint32_t lane, uint32_t n, uint32_t k, uint32_t i, uint32_t floor) {  // k, i uniform
        const uint32_t p = (uint32_t)__popcll(__ballot(before(k, i)));
        if (p >= n) return;
        const uint32_t pk = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)key, 0x138, 0xf, 0xf, false);  // the lane below's
        const uint32_t pi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)id, 0x138, 0xf, 0xf, false);
        key = lane < p ? key : lane == p ? k : pk;
        id = lane < p ? id : lane == p ? i : pi;
        const uint32_t last = (uint32_t)__builtin_amdgcn_readlane((int)key, (int)(n - 1u));
        least = value_of(last > floor ? last : floor);
    }
    // every lane's value z of id `i` (where ok)
    __device__ __forceinline__ void take(uint32_t lane, uint32_t n, float z, uint32_t i, bool ok, uint32_t floor) {
        uint64_t left = __ballot(ok && !(z < least));
        while (left) {
            const int l = __ffsll((unsigned long long)left) - 1;
            left &= left - 1;
            put(lane, n, (uint32_t)__builtin_amdgcn_readlane((int)ordered(z), l), (uint32_t)__builtin_amdgcn_readlane((int)i, l),
                floor);
        }
    }
};

template <bool BF, bool TOP, bool ENT>
struct Stream {
    static constexpr uint32_t VE = BF ? 8 : 4, U = kPer / VE;
    Sums x{kLowest, 0.f, 0.f};
    Best best;
    uint32_t floor = 0;
    bool fresh = true;
    const uint32_t lane, n;
    __device__ __forceinline__ Stream(uint32_t l, uint32_t n_top) : lane(l), n(n_top) {}
    static __device__ __forceinline__ void open(u32x4 r, float* v) {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            if (BF) {
                v[2 * k] = __uint_as_float(r[k] << 16);
                v[2 * k + 1] = __uint_as_float(r[k] & 0xFFFF0000u);
            } else {
                v[k] = __uint_as_float(r[k]);
            }
        }
    }
    __device__ __forceinline__ void add(const float* v, uint32_t count, float most) {
        const float m = larger(x.m, most);
        x = to_reference(x, m);
#pragma unroll
        for (uint32_t k = 0; k < count; k++) {
            const float d = v[k] - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
            x.s += e;
            if (ENT) x.u = fmaf(e, fmaxf(d, -1e30f), x.u);
        }
    }
    // U vectors of a lane, the first of id `id0`, the others 64 VE ids apart; vectors
    // from `end` ids on do not count (CUT)
    template <bool CUT>
    __device__ __forceinline__ void block(const u32x4 (&raw)[U], uint32_t id0, uint32_t end) {
        float v[kPer], top[U], most = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < U; i++) {
            open(raw[i], v + VE * i);
            const bool ok = !CUT || id0 + 64u * VE * i < end;
            float t = -INFINITY;
#pragma unroll
            for (uint32_t k = 0; k < VE; k++) {
                if (CUT && !ok) v[VE * i + k] = -INFINITY;
                t = larger(t, v[VE * i + k]);
            }
            top[i] = t;
            most = larger(most, t);
        }
        add(v, kPer, most);
        if (!TOP) return;
        if (fresh) {  // the n-th largest of the lanes' largest: at least n values are no less
            fresh = false;
            const uint32_t mine = ordered(most);
            uint32_t rank = 0;
#pragma unroll 8
            for (uint32_t l = 0; l < 64; l++) {
                const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)l);
                rank += o > mine || (o == mine && l < lane) ? 1u : 0u;
            }
            const uint64_t nth = __ballot(rank == n - 1u);
            floor = (uint32_t)__builtin_amdgcn_readlane((int)mine, __ffsll((unsigned long long)nth) - 1);
            best.least = value_of(floor);
        }
#pragma unroll
        for (uint32_t i = 0; i < U; i++) {
            if (!__ballot(!(top[i] < best.least))) continue;
            const uint32_t id = id0 + 64u * VE * i;
#pragma unroll
            for (uint32_t k = 0; k < VE; k++) best.take(lane, n, v[VE * i + k], id + k, !CUT || id < end, floor);
        }
    }
};

template <bool BF, bool TOP, bool ENT>
__global__ __launch_bounds__(256) void logp_part_kernel(Logp p) {
    using St = Stream<BF, TOP, ENT>;
    constexpr uint32_t VE = St::VE, U = St::U, ES = BF ? 2 : 4;
    const uint32_t lane = threadIdx.x & 63u, wave = uni(blockIdx.x * 4u + (threadIdx.x >> 6));
    const uint32_t row = wave / p.parts, part = wave - row * p.parts;
    if (row >= p.a.n_rows) return;
    const uint32_t V = p.a.n_vocab;
    const uint8_t* base = (const uint8_t*)p.a.d_logits + (uint64_t)row * p.a.stride * ES;
    // whole 16 bytes from the first aligned value on; what is before and behind them is
    // the first part's
    const uint32_t off = (uint32_t)((0u - (uint32_t)(uintptr_t)base) & 15u) / ES, head = off < V ? off : V;
    const uint32_t nv = (V - head) / VE, tail = head + nv * VE;
    const uint32_t v0 = (uint32_t)((uint64_t)nv * part / p.parts), v1 = (uint32_t)((uint64_t)nv * (part + 1u) / p.parts);
    St st(lane, p.a.n_top);
    const rsrc_t rs = make_rsrc(base + (uint64_t)head * ES, nv * 16u);
    auto load = [&](u32x4 (&raw)[U], uint32_t v) {
#pragma unroll
        for (uint32_t i = 0; i < U; i++) raw[i] = bld16_nt(rs, (v + 64u * i + lane) * 16u, 0);
    };
    uint32_t v = v0;
    const uint32_t end = head + v1 * VE;
    u32x4 a[U], b[U];
    if (v < v1) load(a, v);
    while (v < v1) {
        const uint32_t next = v + 64u * U;
        if (next < v1) load(b, next);
        if (next <= v1) st.template block<false>(a, head + (v + lane) * VE, end);
        else st.template block<true>(a, head + (v + lane) * VE, end);
        v = next;
#pragma unroll
        for (uint32_t i = 0; i < U; i++) a[i] = b[i];
    }
    if (part == 0 && head + (V - tail) > 0) {
        const uint32_t id = lane < head ? lane : tail + lane - head;
        const bool ok = id < V;
        float z = -INFINITY;
        if (ok) z = BF ? bf2f(gld((const uint16_t*)base + id)) : gld((const float*)base + id);
        st.add(&z, 1, z);
        if (TOP) st.best.take(lane, p.a.n_top, z, id, ok, st.floor);
    }
    const Sums x = wave_join(st.x);
    const uint64_t slot = (uint64_t)row * p.parts + part;
    if (lane == 0) gst((f32x4*)(p.sums + 4u * slot), f32x4{x.m, x.s, x.u, 0.f});
    if (TOP && lane < p.a.n_top) {
        uint32_t* o = p.top + 2u * (slot * p.a.n_top + lane);
        gst((u32x2*)o, u32x2{st.best.key, st.best.id});
    }
}

WL_DEV Sums row_sums(const Logp& p, uint32_t row, uint32_t lane) {
    Sums x{kLowest, 0.f, 0.f};
    for (uint32_t i = lane; i < p.parts; i += 64u) {
        const f32x4 v = gld((const f32x4*)(p.sums + 4u * ((uint64_t)row * p.parts + i)));
        x = join(x, Sums{v[0], v[1], v[2]});
    }
    return wave_join(x);
}

// Work-groups [0, rows): a row's entropy and most likely tokens; behind them a wave a token.
template <bool BF>
__global__ __launch_bounds__(256) void logp_join_kernel(Logp p, uint32_t rows) {
    __shared__ u32x2 lists[4][WL_LOGPROB_MAX_TOP];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = uni(tid >> 6), n = p.a.n_top;
    if (blockIdx.x >= rows) {
        const uint32_t t = (blockIdx.x - rows) * 4u + wv;
        if (t >= p.a.n_tokens) return;
        const int32_t token = p.a.d_token[t], row = p.a.d_row ? p.a.d_row[t] : (int32_t)t;
        const bool ok = token >= 0 && (uint32_t)token < p.a.n_vocab && row >= 0 && (uint32_t)row < p.a.n_rows;
        float z = __builtin_nanf("");
        if (ok) {
            const uint64_t at = (uint64_t)(uint32_t)row * p.a.stride + (uint32_t)token;
            z = BF ? bf2f(gld((const uint16_t*)p.a.d_logits + at)) : gld((const float*)p.a.d_logits + at);
            const Sums x = row_sums(p, (uint32_t)row, lane);
            z = (z - x.m) - logf(x.s);
        } else if (lane == 0) {
            set_status(p.a.d_status, WL_PAGED_E_SLOT);
        }
        if (lane == 0) gst(p.a.d_logp + t, z);
        return;
    }
    const uint32_t row = blockIdx.x;
    const Sums x = row_sums(p, row, lane);
    const float log_s = logf(x.s);
    if (tid == 0 && p.a.d_entropy) gst(p.a.d_entropy + row, log_s - x.u / x.s);
    if (n == 0) return;
    // the parts' lists, dealt out to the waves, then the waves' to the first
    Best best;
    const uint32_t all = p.parts * n;
    const u32x2* top = (const u32x2*)(p.top + 2ull * row * all);
    for (uint32_t i = 64u * wv; i < all; i += 256u) {
        const bool ok = i + lane < all;
        u32x2 c = {0u, ~0u};
        if (ok) c = gld(top + i + lane);
        best.take(lane, n, value_of(c[0]), c[1], ok && c[0] != 0u, 0u);
    }
    if (lane < n) lists[wv][lane] = u32x2{best.key, best.id};
    __syncthreads();
    if (wv != 0) return;
    for (uint32_t w = 1; w < 4; w++) {
        const u32x2 c = lane < n ? lists[w][lane] : u32x2{0u, ~0u};
        best.take(lane, n, value_of(c[0]), c[1], c[0] != 0u, 0u);
    }
    if (lane < n) {
        gst(p.a.d_top_id + (uint64_t)row * n + lane, (int32_t)best.id);
        gst(p.a.d_top_logp + (uint64_t)row * n + lane, (value_of(best.key) - x.m) - log_s);
    }
}

// Parts of a row: waves for the whole chip where there are few rows, and no part
// shorter than what a wave has at a time.
uint32_t parts_of(const wl_logprobs& a) {
    const uint32_t most = (a.n_vocab + kPart - 1u) / kPart, want = a.n_rows >= 4096u ? 1u : 4096u / (a.n_rows ? a.n_rows : 1u);
    return want < most ? want : most;
}

}  // namespace

size_t logprobs_scratch(const wl_logprobs& a) {
    const size_t slots = (size_t)(a.n_rows ? a.n_rows : 1) * parts_of(a);
    return slots * (16 + 8 * (size_t)a.n_top);
}

int launch_logprobs(const wl_logprobs& a, void* stream) {
    Logp p{};
    p.a = a;
    p.parts = parts_of(a);
    p.sums = (float*)a.d_scratch;
    p.top = (uint32_t*)(p.sums + 4 * (size_t)a.n_rows * p.parts);
    hipStream_t st = (hipStream_t)stream;
    const bool bf = a.dtype == WL_TYPE_BF16;
    const dim3 grid((uint32_t)(((uint64_t)a.n_rows * p.parts + 3u) / 4u));
    auto part = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p); };
    if (a.n_top && a.d_entropy) bf ? part(logp_part_kernel<true, true, true>) : part(logp_part_kernel<false, true, true>);
    else if (a.n_top) bf ? part(logp_part_kernel<true, true, false>) : part(logp_part_kernel<false, true, false>);
    else if (a.d_entropy) bf ? part(logp_part_kernel<true, false, true>) : part(logp_part_kernel<false, false, true>);
    else bf ? part(logp_part_kernel<true, false, false>) : part(logp_part_kernel<false, false, false>);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    const uint32_t rows = a.d_entropy || a.n_top ? a.n_rows : 0u, wgs = rows + (a.n_tokens + 3u) / 4u;
    if (wgs == 0) return 0;
    if (bf) hipLaunchKernelGGL(logp_join_kernel<true>, dim3(wgs), dim3(256), 0, st, p, rows);
    else hipLaunchKernelGGL(logp_join_kernel<false>, dim3(wgs), dim3(256), 0, st, p, rows);
    return (int)hipGetLastError();
}

}  // namespace paged
}  // namespace wl
