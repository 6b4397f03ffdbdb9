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
// time, their largest, and its own m, s and u, brought to a new m once for the 32. Second
// launch: a work-group a row joins its parts, a wave a token looks up its logit.
//
// The n_top most likely: the first launch leaves the largest value that each lane has met
// (one comparison in 32 values). The n-th largest of these, over the lanes of all parts, is
// a bound that at least n values reach and few others: the second launch finds it, reads
// again what the lanes that reach it have met, and what reaches it too goes into lists in
// LDS, ordered by counting. Where more than kLanes lanes reach the bound (rows of equal
// values, or of -infinity where a grammar leaves fewer than n_top) the whole row is read
// again; a list that runs full is cut down to its n best, and from then on only what is
// before the last of them, by value or by id, comes in. (284 rows of 154880 bf16 with 8 finite
// values, n_top 20: 89 us, one row 63; with equal values coming in whatever their ids,
// a cut at every step, 1069 and 1025.)
//
// Where rows are many f32 is bound by the read of the logits and bf16 by vector operations:
// 12.4 a value (8.5 million instructions of a wave counted for 44 million values), 4 clocks
// each and an exponential 16, some 41 of the 44 thousand clocks of a CU. Where rows are few, two launches.
// 284 rows of 154880: f32 30 us (5.8 TB/s) with no n_top, 42 with 20; bf16 22 us (4.1 TB/s)
// and 31 to 33 (cards differ). One row of them 9 us and 13. 2048 rows of 32000
// bf16: 30 to 32 us and 50. (Lists kept in the first launch, by insertion into each lane's
// registers: 57 us at 284 rows bf16 and n_top 20, 31 at one row.)
constexpr uint32_t kPer = 32;             // values a lane has at a time
constexpr uint32_t kPart = 64 * kPer;     // of a wave
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504088896340736f;

struct Logp {
    wl_logprobs a;
    uint32_t parts;   // per row
    float* sums;      // [n_rows][parts][4] m, s, u
    float* most;      // [n_rows][parts][64] the largest value of each lane
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

// A wave's list of the values that may be among the n largest, of (ordered value, id).
constexpr uint32_t kList = 640;
constexpr uint32_t kLanes = 256;  // whose values are read again
constexpr uint32_t kAhead = 4;    // loads in flight
// Lanes' largest values that a thread holds in registers from its first look at them to its
// second, those behind them it reads again: 80 parts, which a row of 163840 values has where it
// is alone. With 20 and 32 of them, bf16, n_top 20: one row of 154880 13.1 and 13.6 us, of 200003
// 15.0 and 14.2, of 262144 18.1 and 14.7, of 2^20 61 and 57; 2048 rows of 32000, of
// which a thread has one, 50.4 and 52.6 (registers).
constexpr uint32_t kShare = 20;

struct List {
    u32x2* const at;         // [kList] in LDS
    const uint32_t lane, n;
    uint32_t count = 0;
    uint64_t floor = 0;      // what comes in has a place above this
    __device__ __forceinline__ List(u32x2* a, uint32_t l, uint32_t n_top) : at(a), lane(l), n(n_top) {}
    // An ordered value and its id as one number, that of what is before others the larger one.
    static __device__ __forceinline__ uint64_t place(uint32_t k, uint32_t i) { return (uint64_t)k << 32 | ~i; }
    static __device__ __forceinline__ bool before(uint32_t k, uint32_t i, uint32_t k2, uint32_t i2) { return k > k2 || (k == k2 && i < i2); }
    // From four values a lane (0: none): the n-th largest of them, to 16 bits, from below. (A
    // NaN's bound, to 16 bits, is one too.)
    __device__ __forceinline__ void bound(u32x4 mine) {
        uint32_t f = 0;
#pragma unroll
        for (uint32_t b = 31; b >= 16; b--) {
            const uint32_t c = f | 1u << b;
            uint32_t reach = 0;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) reach += (uint32_t)__popcll(__ballot(mine[k] >= c));
            if (reach >= n) f = c;
        }
        floor = ((uint64_t)uni(f) << 32) - (f ? 1u : 0u);
    }
    // Leaves the n best, in order.
    __device__ __forceinline__ void cut() {
        uint32_t k[kList / 64], id[kList / 64], bk = 0, bi = ~0u;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t j = 0; j < kList / 64; j++) {
            const u32x2 x = 64u * j + lane < count ? at[64u * j + lane] : u32x2{0u, ~0u};
            k[j] = x[0];
            id[j] = x[1];
        }
        const uint32_t m = count < n ? count : n;
        for (uint32_t r = 0; r < m; r++) {
            uint32_t x = 0, i = ~0u;
#pragma unroll
            for (uint32_t j = 0; j < kList / 64; j++)
                if (before(k[j], id[j], x, i)) {
                    x = k[j];
                    i = id[j];
                }
            for (int o = 32; o > 0; o >>= 1) {
                const uint32_t x2 = __shfl_xor(x, o, 64), i2 = __shfl_xor(i, o, 64);
                if (before(x2, i2, x, i)) {
                    x = x2;
                    i = i2;
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < kList / 64; j++)
                if (id[j] == i) k[j] = 0, id[j] = ~0u;  // (an id stands in a list once)
            if (lane == r) {
                bk = x;
                bi = i;
            }
        }
        if (lane < m) at[lane] = u32x2{bk, bi};
        __builtin_amdgcn_wave_barrier();
        count = m;
        if (m < n) return;
        floor = place((uint32_t)__builtin_amdgcn_readlane((int)bk, (int)(n - 1u)), (uint32_t)__builtin_amdgcn_readlane((int)bi, (int)(n - 1u)));
    }
    // every lane's value o (ordered) of id i, where ok
    __device__ __forceinline__ void add(uint32_t o, uint32_t i, bool ok) {
        ok = ok && place(o, i) > floor;
        const uint64_t m = __ballot(ok);
        if (!m) return;
        if (ok) at[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u))] = u32x2{o, i};
        count += (uint32_t)__popcll(m);
    }
    // before `more` values a lane come
    __device__ __forceinline__ void make_room(uint32_t more) {
        if (__builtin_expect(count > kList - 64u * more, 0)) cut();
    }
};

template <bool BF, bool TOP, bool ENT>
struct Stream {
    static constexpr uint32_t VE = BF ? 8 : 4, U = kPer / VE;
    Sums x{kLowest, 0.f, 0.f};
    float largest = -INFINITY;  // of this lane
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
        float s = 0.f, u = 0.f;  // (added up by themselves first, 32 values lose less)
#pragma unroll
        for (uint32_t k = 0; k < count; k++) {
            const float d = v[k] - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
            s = k ? s + e : e;
            if (ENT) u = k ? fmaf(e, fmaxf(d, -1e30f), u) : e * fmaxf(d, -1e30f);
        }
        x.s += s;
        if (ENT) x.u += u;
    }
    // U vectors of a lane, 64 apart, of which those before `count` count (CUT)
    template <bool CUT>
    __device__ __forceinline__ void block(const u32x4 (&raw)[U], uint32_t first, uint32_t count) {
        float v[kPer], most = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < U; i++) {
            open(raw[i], v + VE * i);
#pragma unroll
            for (uint32_t k = 0; k < VE; k++) {
                if (CUT && first + 64u * i >= count) v[VE * i + k] = -INFINITY;
                most = larger(most, v[VE * i + k]);
            }
        }
        add(v, kPer, most);
        if (TOP) largest = larger(largest, most);
    }
};

// A row's 16-byte vectors: the first value of vector 0, and how many there are. What is
// before and behind them is the first part's.
template <bool BF>
struct Row {
    static constexpr uint32_t VE = BF ? 8 : 4, ES = BF ? 2 : 4;
    const uint8_t* base;
    uint32_t head, nv, tail;
    __device__ __forceinline__ Row(const Logp& p, uint32_t row) {
        base = (const uint8_t*)p.a.d_logits + (uint64_t)row * p.a.stride * ES;
        const uint32_t off = (uint32_t)((0u - (uint32_t)(uintptr_t)base) & 15u) / ES;
        head = off < p.a.n_vocab ? off : p.a.n_vocab;
        nv = (p.a.n_vocab - head) / VE;
        tail = head + nv * VE;
    }
    __device__ __forceinline__ uint32_t part_at(const Logp& p, uint32_t part) const { return (uint32_t)((uint64_t)nv * part / p.parts); }
    __device__ __forceinline__ float value(uint32_t id) const {
        return BF ? bf2f(gld((const uint16_t*)base + id)) : gld((const float*)base + id);
    }
    // the value before or behind the vectors that a lane has (of id < n_vocab)
    __device__ __forceinline__ uint32_t edge(uint32_t lane) const { return lane < head ? lane : tail + lane - head; }
};

template <bool BF, bool TOP, bool ENT>
__global__ __launch_bounds__(256) void logp_part_kernel(Logp p) {
    using St = Stream<BF, TOP, ENT>;
    constexpr uint32_t U = St::U;
    const uint32_t lane = threadIdx.x & 63u, wave = uni(blockIdx.x * 4u + (threadIdx.x >> 6));
    const uint32_t row = wave / p.parts, part = wave - row * p.parts;
    if (row >= p.a.n_rows) return;
    const Row<BF> r(p, row);
    const uint32_t v0 = r.part_at(p, part), v1 = r.part_at(p, part + 1u);
    St st;
    const rsrc_t rs = make_rsrc(r.base + (uint64_t)r.head * Row<BF>::ES, r.nv * 16u);
    auto load = [&](u32x4 (&raw)[U], uint32_t v) {
#pragma unroll
        for (uint32_t i = 0; i < U; i++) raw[i] = bld16_nt(rs, (v + 64u * i + lane) * 16u, 0);
    };
    uint32_t v = v0;
    u32x4 a[U], b[U];
    if (v < v1) load(a, v);
    while (v < v1) {
        const uint32_t next = v + 64u * U;
        if (next < v1) load(b, next);
        if (next <= v1) st.template block<false>(a, v + lane, v1);
        else st.template block<true>(a, v + lane, v1);
        v = next;
#pragma unroll
        for (uint32_t i = 0; i < U; i++) a[i] = b[i];
    }
    if (part == 0 && r.head + (p.a.n_vocab - r.tail) > 0) {
        const uint32_t id = r.edge(lane);
        const float z = id < p.a.n_vocab ? r.value(id) : -INFINITY;
        st.add(&z, 1, z);
    }
    const Sums x = wave_join(st.x);
    const uint64_t slot = (uint64_t)row * p.parts + part;
    if (lane == 0) gst((f32x4*)(p.sums + 4u * slot), f32x4{x.m, x.s, x.u, 0.f});
    if (TOP) gst(p.most + 64u * slot + lane, st.largest);
}

// Part i's m, s and u (behind the last part: the last one's, taken away by row_sums).
WL_DEV f32x4 part_sums(const Logp& p, uint32_t row, uint32_t i) {
    return gld((const f32x4*)(p.sums + 4u * ((uint64_t)row * p.parts + (i < p.parts ? i : p.parts - 1u))));
}
// All parts', of which the lane has part `lane` already.
WL_DEV Sums row_sums(const Logp& p, uint32_t row, uint32_t lane, f32x4 v) {
    Sums x{kLowest, 0.f, 0.f};
    if (lane < p.parts) x = Sums{v[0], v[1], v[2]};
    for (uint32_t i = lane + 64u; i < p.parts; i += 64u) {
        v = part_sums(p, row, i);
        x = join(x, Sums{v[0], v[1], v[2]});
    }
    return wave_join(x);
}

// Work-groups [0, rows): a row's entropy and most likely tokens; behind them a wave a token.
template <bool BF>
__global__ __launch_bounds__(256) void logp_join_kernel(Logp p, uint32_t rows) {
    constexpr uint32_t VE = Row<BF>::VE;
    __shared__ u32x2 lists[4][kList];
    __shared__ uint32_t lanes[kLanes];  // those whose largest reach the bound
    __shared__ u32x4 highs[64];
    __shared__ uint32_t n_lanes, counts[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = uni(tid >> 6), n = p.a.n_top;
    if (blockIdx.x >= rows) {
        const uint32_t t = (blockIdx.x - rows) * 4u + wv;
        if (t >= p.a.n_tokens) return;
        const int32_t token = p.a.d_token[t], row = p.a.d_row ? p.a.d_row[t] : (int32_t)t;
        if (token == -1) return;
        const bool ok = token >= 0 && (uint32_t)token < p.a.n_vocab && row >= 0 && (uint32_t)row < p.a.n_rows;
        float z = __builtin_nanf("");
        if (ok) {
            const uint64_t at = (uint64_t)(uint32_t)row * p.a.stride + (uint32_t)token;
            z = BF ? bf2f(gld((const uint16_t*)p.a.d_logits + at)) : gld((const float*)p.a.d_logits + at);
            const Sums x = row_sums(p, (uint32_t)row, lane, part_sums(p, (uint32_t)row, lane));
            z = (z - x.m) - logf(x.s);
        } else if (lane == 0) {
            set_status(p.a.d_status, WL_PAGED_E_SLOT);
        }
        if (lane == 0) gst(p.a.d_logp + t, z);
        return;
    }
    const uint32_t row = blockIdx.x;
    const f32x4 first = part_sums(p, row, lane);
    const uint32_t all = 64u * p.parts;  // lanes
    const float* most = p.most + 64ull * row * p.parts;
    float share[kShare];  // of their largest values
    if (n) {
#pragma unroll
        for (uint32_t k = 0; k < kShare; k++)
            if (256u * k < all) share[k] = gld(most + (tid + 256u * k < all ? tid + 256u * k : lane));
    }
    const Sums x = row_sums(p, row, lane, first);
    const float log_s = logf(x.s);
    if (tid == 0 && p.a.d_entropy) gst(p.a.d_entropy + row, log_s - x.u / x.s);
    if (n == 0) return;
    // a bound from the largest values of the lanes, a share of them to a thread
    List list(lists[wv], lane, n);
    auto shares = [&](auto&& f) {
#pragma unroll
        for (uint32_t k = 0; k < kShare; k++)
            if (tid + 256u * k < all) f(ordered(share[k]), tid + 256u * k);
        for (uint32_t i = tid + 256u * kShare; i < all; i += 256u) f(ordered(gld(most + i)), i);
    };
    uint32_t high = 0;
    shares([&](uint32_t o, uint32_t) { high = max(high, o); });
    ((uint32_t*)highs)[tid] = high;
    if (tid == 0) n_lanes = 0;
    __syncthreads();
    list.bound(highs[lane]);
    shares([&](uint32_t o, uint32_t i) {
        if (List::place(o, 0u) <= list.floor) return;
        const uint32_t k = atomicAdd(&n_lanes, 1u);  // (their order changes no result)
        if (k < kLanes) lanes[k] = i;
    });
    __syncthreads();
    const uint32_t found = uni(n_lanes);
    const bool whole = found > kLanes;
    // what these lanes have met, or the whole row: 64 vectors, one a lane, make a step
    const Row<BF> r(p, row);
    const rsrc_t rs = make_rsrc(r.base + (uint64_t)r.head * Row<BF>::ES, r.nv * 16u);
    const uint32_t each = (r.nv / p.parts + 64u) / 64u;  // vectors of a lane, at most
    const uint32_t sh = each > 1u ? 32u - (uint32_t)__builtin_clz(each - 1u) : 0u;
    const uint32_t steps = ((whole ? r.nv : found << sh) + 63u) / 64u;
    for (uint32_t i0 = wv; i0 < steps; i0 += 4u * kAhead) {
        u32x4 raw[kAhead];
        uint32_t at[kAhead];  // the lane's vector (from nv on: none)
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const uint32_t i = 64u * (i0 + 4u * k) + lane;
            at[k] = ~0u;
            if (whole) {
                at[k] = i;
            } else if (i >> sh < found) {
                const uint32_t x = lanes[i >> sh], v = r.part_at(p, x / 64u) + x % 64u + 64u * (i & ((1u << sh) - 1u));
                if (v < r.part_at(p, x / 64u + 1u)) at[k] = v;
            }
            raw[k] = bld16(rs, at[k] < r.nv ? at[k] * 16u : kOOB, 0);
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            float v[VE];
            Stream<BF, true, true>::open(raw[k], v);
            list.make_room(VE);
#pragma unroll
            for (uint32_t e = 0; e < VE; e++) list.add(ordered(v[e]), r.head + at[k] * VE + e, at[k] < r.nv);
        }
    }
    if (wv == 0) {
        const uint32_t id = r.edge(lane);
        const bool ok = id < p.a.n_vocab && lane < 32u;
        list.make_room(1);
        list.add(ordered(ok ? r.value(id) : 0.f), id, ok);
    }
    // the waves' lists as one, ordered by counting
    if (list.count > 64u) list.cut();
    const u32x2 own = lane < list.count ? lists[wv][lane] : u32x2{0u, ~0u};
    if (lane == 0) counts[wv] = list.count;
    __syncthreads();
    uint32_t before = 0, count = 0;
    for (uint32_t w = 0; w < 4; w++) {
        if (w < wv) before += counts[w];
        count += counts[w];
    }
    u32x2* const one = lists[0];  // at most 256, and zeros up to a multiple of 8
    if (lane < list.count) one[before + lane] = own;
    if (tid < 8u) one[count + tid] = u32x2{0u, ~0u};
    __syncthreads();
    if (lane >= list.count) return;
    uint32_t rank = 0;
    for (uint32_t i = 0; i < count; i += 8u)
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) rank += List::before(one[i + k][0], one[i + k][1], own[0], own[1]) ? 1u : 0u;
    if (rank < n) {
        gst(p.a.d_top_id + (uint64_t)row * n + rank, (int32_t)own[1]);
        gst(p.a.d_top_logp + (uint64_t)row * n + rank, (value_of(own[0]) - x.m) - log_s);
    }
}

// Parts of a row: waves for the whole chip where there are few rows, and no part shorter
// than what a wave has at a time. With n_top more and shorter parts: there is less to read
// again, which outweighs the longer join (in us at 2048, 4096 and 8192 waves, bf16 and n_top
// 20: 284 x 154880 33.0, 31.2, 30.7, 2048 x 32000 62.9, 53.6, 46.7; without n_top 22.2, 22.8,
// 22.9 and 32.7, 32.8, 32.4; 1024 waves 33.3 at the former).
struct Split {
    uint32_t waves, most;  // of the launch where rows are few; parts of a row at the most
};
Split split_of(const wl_logprobs& a) { return Split{a.n_top ? 8192u : 2048u, (a.n_vocab + kPart - 1u) / kPart}; }
uint32_t parts_of(const wl_logprobs& a) {
    const Split s = split_of(a);
    const uint32_t want = a.n_rows >= s.waves ? 1u : s.waves / (a.n_rows ? a.n_rows : 1u);
    return want < s.most ? want : s.most;
}

}  // namespace

// Bytes for n_rows x parts_of(a) parts, rounded up to what no call of fewer rows, values or
// alternatives exceeds: fewer rows may come in more parts in all (284 rows 28 each, 256 rows 32).
size_t logprobs_scratch(const wl_logprobs& a) {
    const Split s = split_of(a);
    const size_t rows = a.n_rows ? a.n_rows : 1, all = rows * s.most, few = all < s.waves ? all : s.waves;
    return (rows > few ? rows : few) * (16 + (a.n_top ? 256 : 0));
}

int launch_logprobs(const wl_logprobs& a, void* stream) {
    Logp p{};
    p.a = a;
    p.parts = parts_of(a);
    p.sums = (float*)a.d_scratch;
    p.most = p.sums + 4 * (size_t)a.n_rows * p.parts;
    const uint32_t rows = a.d_entropy || a.n_top ? a.n_rows : 0u, wgs = rows + (a.n_tokens + 3u) / 4u;
    if (wgs == 0) return 0;
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
    if (bf) hipLaunchKernelGGL(logp_join_kernel<true>, dim3(wgs), dim3(256), 0, st, p, rows);
    else hipLaunchKernelGGL(logp_join_kernel<false>, dim3(wgs), dim3(256), 0, st, p, rows);
    return (int)hipGetLastError();
}

}  // namespace paged
}  // namespace wl
