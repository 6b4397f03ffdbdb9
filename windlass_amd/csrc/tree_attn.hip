// tree_attn.hip — attention of trees of drafted tokens over a paged cache of
// latent rows (wl_paged_tree_attention).
#include <hip/hip_runtime.h>

#include "dev_common.h"
#include "paged.h"

namespace wl {
namespace paged {
namespace {

constexpr uint32_t kKT = 64;    // keys of a tile
constexpr uint32_t kGrid = 256; // work-groups of a launch: one per CU (LDS and registers allow one)
constexpr float kNone = -3.0e38f;  // the running maximum of a row that has seen no key

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
#define WL_LDS(p) ((__attribute__((address_space(3))) void*)(p))

// What a launch needs beside the call's arguments.
struct Tree {
    wl_tree_attn a;
    uint32_t psh;      // log2 page_size
    float scale2;      // scale * log2(e): scores in powers of two
    float* part;       // [2 kGrid][rows][cols] unnormalised sums of split tiles
    float* part_ml;    // [2 kGrid][rows][2] their maxima and weight sums
    uint32_t* desc;    // [2 kGrid][4] split tiles: {request + 1, row tile, first and last work-group}
};

// ---- the work and its split --------------------------------------------------
// A request's rows (node, head) come in tiles of ROWS, its keys in tiles of
// kKT; a unit is one of each. The units of all requests, row tile by row tile,
// stand in one row, and work-group c takes [c per, c per + per) of them, so
// every work-group has the same number of key tiles to go through, whatever
// the requests' lengths. A row tile that falls into one work-group is finished
// there; one that is split leaves its parts in the scratch for the second
// launch. Work-group b runs on XCD b % 8: c = (b % 8)(G / 8) + b / 8, so the
// row tiles of a request that run at the same time share one XCD's L2.
struct Req {
    uint32_t t0, nodes, len, keys, nrt, nkt, flaw;  // flaw: WL_PAGED_E_* (its rows get NaN)
};
template <uint32_t ROWS>
WL_DEV Req request(const Tree& p, uint32_t r, uint32_t& status) {
    Req q{};
    const int32_t t0 = p.a.d_cu[r], t1 = p.a.d_cu[r + 1], n = p.a.d_len[r];
    if (t0 < 0 || t1 < t0 || (uint32_t)t1 > p.a.n_tokens) {
        status |= WL_PAGED_E_LEN;
        return q;
    }
    q.t0 = (uint32_t)t0;
    q.nodes = (uint32_t)(t1 - t0);
    if (q.nodes == 0) return q;
    if (n < 0 || (uint64_t)(uint32_t)n + q.nodes > ((uint64_t)p.a.max_pages << p.psh)) q.flaw |= WL_PAGED_E_LEN;
    if (q.nodes > WL_TREE_MAX_NODES) q.flaw |= WL_PAGED_E_TREE;
    status |= q.flaw;
    q.len = (uint32_t)n;
    q.keys = q.len + q.nodes;
    q.nrt = (q.nodes * p.a.n_heads + ROWS - 1) / ROWS;
    q.nkt = q.flaw ? 1u : (q.keys + kKT - 1) / kKT;
    return q;
}

// The launch's units, and the request (and its first unit) that unit u0 = c per
// falls into. Each thread sums the requests of its share; tmp: a word per wave, and two.
struct Place {
    uint64_t total, per, u0, base;
    uint32_t r;
};
template <uint32_t ROWS, uint32_t THREADS>
WL_DEV Place find_place(const Tree& p, uint32_t c, uint32_t min_per, uint64_t* tmp) {
    constexpr uint32_t NW = THREADS / 64;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6, R = p.a.n_req;
    const uint32_t share = (R + THREADS - 1u) / THREADS;
    uint64_t mine = 0;
    uint32_t status = 0;
    for (uint32_t i = 0; i < share; i++) {
        const uint32_t r = tid * share + i;
        if (r < R) {
            const Req q = request<ROWS>(p, r, status);
            mine += (uint64_t)q.nrt * q.nkt;
        }
    }
    if (c == 0 && status && p.a.d_status)
        __hip_atomic_fetch_or(p.a.d_status, status, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    uint64_t inc = mine;
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint64_t v = (uint64_t)__shfl_up((unsigned long long)inc, o, 64);
        if (lane >= o) inc += v;
    }
    if (lane == 63) tmp[wv] = inc;
    __syncthreads();
    Place f;
    f.total = 0;
#pragma unroll
    for (uint32_t w = 0; w < NW; w++) f.total += tmp[w];
    f.per = (f.total + kGrid - 1) / kGrid;
    if (f.per < min_per) f.per = min_per;
    f.u0 = (uint64_t)c * f.per;
    uint64_t at = inc - mine;
    for (uint32_t w = 0; w < wv; w++) at += tmp[w];
    if (f.u0 >= at && f.u0 < at + mine) {  // one thread at most
        for (uint32_t i = 0; i < share; i++) {
            const uint32_t r = tid * share + i;
            const Req q = request<ROWS>(p, r, status);
            const uint64_t n = (uint64_t)q.nrt * q.nkt;
            if (f.u0 < at + n) {
                tmp[NW] = at;
                tmp[NW + 1] = r;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    f.base = tmp[NW];
    f.r = uni((uint32_t)tmp[NW + 1]);
    __syncthreads();
    return f;
}

__device__ const uint32_t g_zero[4] = {0u, 0u, 0u, 0u};

WL_DEV uint32_t pack_bf16(float a, float b) {
    bf16x2 r;
    r[0] = (__bf16)a;  // round to nearest even
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
}
WL_DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
WL_DEV bool has_nonfinite(u32x4 v) {
    bool f = false;
#pragma unroll
    for (int i = 0; i < 4; i++)
        f |= (v[i] & 0x7F80u) == 0x7F80u || (v[i] & 0x7F800000u) == 0x7F800000u;
    return f;
}
// Where a row's 16-byte chunks lie in LDS: chunk c at c ^ swz(row) (rows of 256
// bytes or more) or c ^ swz8(row) (rows of 128). LDS serves a 16-byte read 16
// lanes at a time, lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 of either
// half wave: for an MFMA operand (lane = row + 16 x chunk) those are 8 rows at
// an even chunk and the other 8 at the odd one beside it, which these put into
// 16 different places of the 256 bytes that the banks cover. A transposing
// read's 32 lanes (8 rows x 2 chunks) fall into 16 different ones too.
// Measured: 237 bytes a clock and CU, 127 with a swizzle over 16 rows in order.
WL_DEV constexpr uint32_t swz(uint32_t row) { return ((row & 3u) << 1) | (row & 8u); }
WL_DEV constexpr uint32_t swz8(uint32_t row) { return (row & 2u) | ((row & 8u) >> 1); }

// ---- 16-bit queries and cache --------------------------------------------------
// ROWS = 16 MT RG rows (node, head) against 64 keys at a time, RG groups of four
// waves with 16 MT rows each.
//   S^T[keys][rows] = K Q^T: wave (ks, kh) of a group takes keys [32 ks, + 32)
//           and half kh of the columns (of the latent and of the rotary ones),
//           whose part of the queries it holds in registers (2 LC + 1 steps of
//           32 columns, MT row tiles) through the whole walk; it hands the sums of one 16-key tile to the wave of the
//           other half and takes those of its own, 16 (2 ks + kh), from it;
//   P = 2^(S - m) in bf16, through LDS, to all waves of the group;
//   O^T[cols][rows] += V^T P^T: wave w owns columns [32 LC w, + 32 LC); the key
//           rows are read again, transposed (ds_read_b64_tr_b16).
// m is a reference, not the maximum: that of the walk's first tile. Weights may
// exceed 1 and lose nothing by it (bf16 and f32 keep their relative precision);
// only where a score passes it by kSlack powers of two the walk is done again,
// after one over the scores alone for the true maxima. So nothing is rescaled,
// and a tile costs three barriers.
// Key rows come into LDS by DMA (16 bytes a lane), a tile ahead, a wave for a
// row, its address in scalars: rows behind the last key and columns behind the
// row's are read as zeros by the resource's bounds. The rotary parts have one
// buffer, filled again as soon as the scores are there.
constexpr float kSlack = 64.f;  // a weight at most 2^64, 2^31 of them 2^95

template <int MT, int RG, int LC>
__global__ __launch_bounds__(256 * RG) void tree_bf16_kernel(Tree p, uint32_t min_per) {
    constexpr uint32_t ROWS = 16 * MT * RG, PITCH = 256 * LC, NL = 2 * LC, NS = NL + 1, CT = 2 * LC, DR = 16 / RG;
    __shared__ __align__(1024) uint8_t lat0[kKT * PITCH], lat1[kKT * PITCH];
    __shared__ __align__(1024) uint8_t rot[kKT * 128];
    // a slot per wave, written by the other half's wave (partial scores) and,
    // once it has read them, by itself: its weights [rows of the group][16 keys]
    // and its rows' maxima
    constexpr uint32_t SLOT = 1024 * MT, MAXIMA = 512 * MT;
    __shared__ __align__(1024) uint8_t xbuf[4 * RG * SLOT];
    __shared__ uint64_t seen[ROWS];
    __shared__ float wsum[4][ROWS];
    __shared__ uint32_t bad_page, again;
    __shared__ uint64_t tmp[4 * RG + 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uni(tid >> 6), n = lane & 15u, g = lane >> 4;
    const uint32_t wv = wave & 3u, kh = wave & 1u, r0 = 16u * MT * (wave >> 2);
    uint8_t* slot_own = xbuf + wave * SLOT;
    uint8_t* slot_other = xbuf + (wave ^ 1u) * SLOT;
    const uint8_t* slots = xbuf + (wave & ~3u) * SLOT;  // the group's
    const uint32_t c = (blockIdx.x % 8u) * (kGrid / 8u) + blockIdx.x / 8u;
    const uint32_t H = p.a.n_heads, L = p.a.cache.kv_lora_rank, RP = p.a.cache.qk_rope;
    if (tid == 0) bad_page = again = 0;
    const Place f = find_place<ROWS, 256 * RG>(p, c, min_per, tmp);
    const uint64_t u1 = f.u0 + f.per < f.total ? f.u0 + f.per : f.total;
    if (tid < 2) p.desc[4 * (2 * c + tid)] = 0;
    if (f.u0 >= u1) return;

    uint64_t u = f.u0, base = f.base;
    uint32_t r = f.r, status = 0;
    Req q = request<ROWS>(p, r, status);
    while (u < u1) {
        while (u >= base + (uint64_t)q.nrt * q.nkt) {  // the next request that has units
            base += (uint64_t)q.nrt * q.nkt;
            q = request<ROWS>(p, ++r, status);
        }
        const uint32_t rt = uni((uint32_t)((u - base) / q.nkt)), kt0 = uni((uint32_t)((u - base) % q.nkt));
        const uint32_t kt1 = uni((uint32_t)(u1 - u < q.nkt - kt0 ? kt0 + (u1 - u) : q.nkt));
        u += kt1 - kt0;
        const uint32_t rows = uni(q.nodes * H - rt * ROWS < ROWS ? q.nodes * H - rt * ROWS : ROWS);
        const int32_t* table = p.a.d_table + (size_t)r * p.a.max_pages;

        f32x4 acc[MT][CT];
        float m[MT], l[MT];
        auto clear = [&]() {
#pragma unroll
            for (int i = 0; i < MT; i++) {
                l[i] = 0.f;
#pragma unroll
                for (uint32_t j = 0; j < CT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        };
        bool bad = false;
        if (q.flaw) {
            clear();
#pragma unroll
            for (int i = 0; i < MT; i++) m[i] = kNone;
        } else {
            int32_t page = 0;
            // the page of key 64 t + lane
            auto page_of = [&](uint32_t t) {
                const uint32_t key = t * kKT + lane;
                return key < q.keys ? table[key >> p.psh] : -1;
            };
            uint32_t ri_rot = 0, nb_rot = 0;
            auto issue = [&](uint8_t* lat, uint32_t t, int32_t page) {
                const uint32_t key = t * kKT + lane;
                const bool ok = key < q.keys && page >= 0 && (uint32_t)page < p.a.cache.n_pages;
                bad |= key < q.keys && !ok;
                const uint32_t ri = ok ? ((uint32_t)page << p.psh) + (key & (p.a.cache.page_size - 1u)) : 0u;
                const uint32_t nb = ok ? 2u * L : 0u;  // a row that is not there is read as zeros
                const uint64_t sb = 2ull * p.a.cache.row_stride;
                uint32_t lx = lane * 16u;
                asm volatile("" : "+v"(lx));  // the offsets are worked out per tile, not held
                const uint32_t d0 = DR * wave;
#pragma unroll
                for (uint32_t i = 0; i < DR; i++) {
                    const uint32_t row = __builtin_amdgcn_readlane(ri, d0 + i);
                    const rsrc_t rs = make_rsrc((const uint8_t*)p.a.cache.d_rows + row * sb, __builtin_amdgcn_readlane(nb, d0 + i));
                    if (LC == 4 || lane < 16 * LC)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, WL_LDS(lat + (d0 + i) * PITCH), 16u,
                                                                 lx ^ (16u * swz((d0 + i) & 15u)), 0u, 0, 0);
                }
                ri_rot = ri;
                nb_rot = nb;
            };
            auto issue_rot = [&]() {
#pragma unroll
                for (uint32_t j = 0; j < DR / 8; j++) {
                    const uint32_t kr = DR * wave + 8u * j + (lane >> 3);
                    const uint32_t row = __shfl(ri_rot, kr, 64), there = __shfl(nb_rot, kr, 64);
                    const uint32_t ch = (lane & 7u) ^ swz8(kr & 15u);
                    const uint8_t* src = there && 8u * ch < RP ? (const uint8_t*)p.a.cache.d_rows +
                                                                     row * (2ull * p.a.cache.row_stride) + 2u * L + 16u * ch
                                                               : (const uint8_t*)g_zero;
                    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)src,
                                                     WL_LDS(rot + (DR * wave + 8u * j) * 128u), 16u, 0, 0);
                }
            };
            // the queries, in the operand's layout: lane (row n, k group g)
            bf16x8 qf[MT][NS];
            const rsrc_t ql = make_rsrc((const uint16_t*)p.a.d_q_lat + q.t0 * p.a.q_lat_stride,
                                        2u * ((q.nodes - 1u) * (uint32_t)p.a.q_lat_stride + H * L));
            const rsrc_t qr = make_rsrc((const uint16_t*)p.a.d_q_rope + q.t0 * p.a.q_rope_stride,
                                        2u * ((q.nodes - 1u) * (uint32_t)p.a.q_rope_stride + H * RP));
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const uint32_t lr = r0 + 16u * i + n, row = rt * ROWS + lr, node = row / H, h = row - node * H;
                const bool live = lr < rows;
                const uint32_t vl = live ? 2u * (node * (uint32_t)p.a.q_lat_stride + h * L + 8u * g) : kOOB;
                const uint32_t vr = live ? 2u * (node * (uint32_t)p.a.q_rope_stride + h * RP + 8u * g) : kOOB;
#pragma unroll
                for (uint32_t s = 0; s < NS; s++) {
                    const bool lat = s < NL;
                    const uint32_t o = 64u * (lat ? kh * NL + s : kh);
                    u32x4 x = lat ? bld16(ql, vl + o, 0) : bld16(qr, vr + o, 0);
                    if (o / 2u + 8u * g >= (lat ? L : RP)) x = u32x4{0u, 0u, 0u, 0u};
                    qf[i][s] = as_bf16x8(x);
                }
                if (wv == 0 && g == 0) {
                    const uint32_t nd = live ? node : 0u;
                    seen[lr] = p.a.d_mask ? p.a.d_mask[q.t0 + nd] : (2ull << nd) - 1ull;
                }
            }
            // the scores of tile t for this wave's 16 keys (row n, keys 4 g + j of them) in
            // powers of two; `between` runs once the rotary buffer is free
            auto scores = [&](uint8_t* lat, uint32_t t, uint32_t lane, f32x4* sc, auto between) {
                const uint32_t n = lane & 15u, g = lane >> 4;
                // this half's part of the scores of keys 32 ks + 16 k + ...: chunk 4 st + g of a
                // row lies at (64 st) ^ (16 (g ^ swz))
                f32x4 pa[2][MT];
#pragma unroll
                for (int i = 0; i < MT; i++) pa[0][i] = pa[1][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                const uint32_t key0 = 32u * (wv >> 1) + n;
                const uint32_t ko = key0 * PITCH, kx = 16u * (g ^ swz(n));
                const uint32_t ro = key0 * 128u + 16u * (g ^ swz8(n));
                auto kread = [&](uint32_t s, uint32_t k) {
                    return s < NL ? *(const u32x4*)(lat + ko + ((64u * (kh * NL + s)) ^ kx) + 16u * k * PITCH)
                                  : *(const u32x4*)(rot + (ro ^ (64u * kh)) + 2048u * k);
                };
                {  // the reads of a step ahead of its products
                    u32x4 kf[2][2];
                    kf[0][0] = kread(0, 0);
                    kf[0][1] = kread(0, 1);
#pragma unroll
                    for (uint32_t s = 0; s < NS; s++) {
                        const uint32_t b = s & 1u;
                        if (s + 1 < NS) {
                            kf[b ^ 1u][0] = kread(s + 1, 0);
                            kf[b ^ 1u][1] = kread(s + 1, 1);
                        }
#pragma unroll
                        for (uint32_t k = 0; k < 2; k++)
#pragma unroll
                            for (int i = 0; i < MT; i++) pa[k][i] = mma(as_bf16x8(kf[b][k]), qf[i][s], pa[k][i]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    *(f32x4*)(slot_other + 1024u * i + 16u * lane) = kh ? pa[0][i] : pa[1][i];
                    sc[i] = kh ? pa[1][i] : pa[0][i];
                }
                lds_barrier();
                between();
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    const f32x4 o = *(const f32x4*)(slot_own + 1024u * i + 16u * lane);
#pragma unroll
                    for (int j = 0; j < 4; j++) sc[i][j] = (kh ? o[j] + sc[i][j] : sc[i][j] + o[j]) * p.scale2;
                }
                if ((t + 1) * kKT > q.len) {  // tree nodes, or the end, in this tile
                    // a row that some nodes may not see must not reach them through
                    // 0 x inf: its non-finite chunks are cleared (every score is
                    // there), and its scores are NaN for those that see it. The
                    // rotary part only enters scores.
                    const uint32_t mykey = t * kKT + 16u * wv + n;
                    uint32_t nf = 0;
                    if (mykey >= q.len) {
                        uint8_t* row = lat + (16u * wv + n) * PITCH + 16u * g;
#pragma unroll 1
                        for (uint32_t s = 0; s < 4 * LC; s++) {
                            u32x4* x = (u32x4*)(row + 64u * s);
                            if (has_nonfinite(*x)) {
                                nf = 1;
                                *x = u32x4{0u, 0u, 0u, 0u};
                            }
                        }
                    }
                    uint64_t fl = __ballot(nf != 0);  // lane 16 g + n: key n
                    fl |= fl >> 32;
                    const uint32_t flawed = (uint32_t)(fl | (fl >> 16));
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t kj = 4u * g + j, key = t * kKT + 16u * wv + kj;
                        const float nan = (flawed >> kj) & 1u ? __builtin_nanf("") : 0.f;
#pragma unroll
                        for (int i = 0; i < MT; i++) {
                            const uint32_t bit = (uint32_t)(seen[r0 + 16u * i + n] >> ((key - q.len) & 63u)) & (key < q.keys ? 1u : 0u);
                            sc[i][j] = (bit | (key < q.len ? 1u : 0u)) ? sc[i][j] + nan : -INFINITY;
                        }
                    }
                }
            };
            // m = the largest of m and what the group's waves have in x (a row's lanes differ in g)
            auto share_maxima = [&](float* x) {
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    x[i] = fmaxf(x[i], __shfl_xor(x[i], 16, 64));
                    x[i] = fmaxf(x[i], __shfl_xor(x[i], 32, 64));
                    if (g == 0) *(float*)(slot_own + MAXIMA + 4u * (16u * i + n)) = x[i];
                }
                lds_barrier();
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    m[i] = kNone;
#pragma unroll
                    for (uint32_t w = 0; w < 4; w++) m[i] = fmaxf(m[i], *(const float*)(slots + w * SLOT + MAXIMA + 4u * (16u * i + n)));
                }
            };
            bool pass = false;
            uint32_t first = kt0;  // the tile that sets the reference
            auto step = [&](uint8_t* lat, uint8_t* nlat, uint32_t t) {
                uint32_t lane = tid & 63u;
                asm volatile("" : "+v"(lane));  // addresses are worked out per tile, not held in registers
                const uint32_t n = lane & 15u, g = lane >> 4;
                vm_drain();
                lds_barrier();
                const bool more = t + 1 < kt1;
                if (more) {
                    issue(nlat, t + 1, page);
                    page = page_of(t + 2);
                }
                f32x4 sc[MT];
                scores(lat, t, lane, sc, [&]() {
                    if (more) issue_rot();
                });
                if (t == first) {
                    float x[MT];
#pragma unroll
                    for (int i = 0; i < MT; i++) x[i] = fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3]));
                    share_maxima(x);
                }
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    float e[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) e[j] = exp2_(sc[i][j] - m[i]);
                    l[i] += (e[0] + e[1]) + (e[2] + e[3]);
                    *(u32x2*)(slot_own + (16u * i + n) * 32u + 8u * g) = u32x2{pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3])};
                    pass |= fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3])) > m[i] + kSlack;
                }
                lds_barrier();
                // O^T += V^T P^T
                const uint32_t vq = (lane & 15u) >> 2, vb = (lane & 3u) >> 1;
                const uint32_t vo = (8u * g + vq) * PITCH + 16u * ((4u * LC * wv + vb) ^ swz((8u * g + vq) & 15u)) + 8u * (lane & 1u);
                auto vfrag = [&](uint32_t i) {  // columns 16 (i % CT) of the wave's, keys 32 (i / CT) + 8 g + [0, 8)
                    const uint8_t* pa = lat + (vo ^ (32u * (i % CT))) + 32u * PITCH * (i / CT);
                    typedef __attribute__((address_space(3))) s16x4 l_s16x4;
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa));
                    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa + 4 * PITCH));
                    const u32x2 xx = __builtin_bit_cast(u32x2, x), yy = __builtin_bit_cast(u32x2, y);
                    return u32x4{xx[0], xx[1], yy[0], yy[1]};
                };
                constexpr uint32_t VG = 2, NV = 2 * CT;
                u32x4 vf[2][VG];
                bf16x8 pf[MT];
#pragma unroll
                for (uint32_t k = 0; k < VG; k++) vf[0][k] = vfrag(k);
#pragma unroll
                for (uint32_t v = 0; v < NV; v += VG) {
                    const uint32_t b = (v / VG) & 1u, kk = v / CT;
                    if (v % CT == 0) {
#pragma unroll
                        for (int i = 0; i < MT; i++)
                            pf[i] = as_bf16x8(*(const u32x4*)(slots + (2u * kk + (g >> 1)) * SLOT + (16u * i + n) * 32u + 16u * (g & 1u)));
                    }
                    if (v + VG < NV) {
#pragma unroll
                        for (uint32_t k = 0; k < VG; k++) vf[b ^ 1u][k] = vfrag(v + VG + k);
                    }
#pragma unroll
                    for (uint32_t k = 0; k < VG; k++)
#pragma unroll
                        for (int i = 0; i < MT; i++) acc[i][(v + k) % CT] = mma(as_bf16x8(vf[b][k]), pf[i], acc[i][(v + k) % CT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            for (;;) {
                clear();
                issue(lat0, kt0, page_of(kt0));
                issue_rot();
                page = page_of(kt0 + 1);
                for (uint32_t t = kt0; t < kt1; t += 2) {
                    step(lat0, lat1, t);
                    if (t + 1 < kt1) step(lat1, lat0, t + 1);
                }
                if (first != kt0) break;
                if (__ballot(pass) && lane == 0) again = 1u;
                lds_barrier();
                const bool redo = again != 0;
                lds_barrier();
                if (!redo) break;
                if (tid == 0) again = 0u;
                float x[MT];
#pragma unroll
                for (int i = 0; i < MT; i++) x[i] = kNone;
                for (uint32_t t = kt0; t < kt1; t++) {
                    issue(lat0, t, page_of(t));
                    issue_rot();
                    vm_drain();
                    lds_barrier();
                    f32x4 sc[MT];
                    scores(lat0, t, lane, sc, [] {});
#pragma unroll
                    for (int i = 0; i < MT; i++)
                        x[i] = fmaxf(x[i], fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3])));
                    lds_barrier();
                }
                share_maxima(x);
                lds_barrier();
                first = ~0u;
            }
        }
        // the weight sums over the waves' keys; flaws
        if (__ballot(bad) && lane == 0) {
            bad_page = 1u;
            if (p.a.d_status)
                __hip_atomic_fetch_or(p.a.d_status, WL_PAGED_E_PAGE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
            l[i] += __shfl_xor(l[i], 16, 64);
            l[i] += __shfl_xor(l[i], 32, 64);
            if (g == 0) wsum[wv][r0 + 16u * i + n] = l[i];
        }
        __syncthreads();
        const bool nan = bad_page != 0 || q.flaw;
        const bool whole = kt0 == 0 && kt1 == q.nkt;
        const uint32_t slot = 2u * c + (kt0 == 0 ? 1u : 0u);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const uint32_t lr = r0 + 16u * i + n;
            float sum = (wsum[0][lr] + wsum[1][lr]) + (wsum[2][lr] + wsum[3][lr]);
            if (nan) sum = __builtin_nanf("");
            if (lr < rows) {
                if (whole) {
                    const uint32_t row = rt * ROWS + lr, node = row / H, h = row - node * H;
                    uint16_t* o = (uint16_t*)p.a.d_out + (size_t)(q.t0 + node) * p.a.out_stride + (size_t)h * L;
                    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
                    for (uint32_t ct = 0; ct < CT; ct++) {
                        const uint32_t col = 32u * LC * wv + 16u * ct + 4u * g;
                        const f32x4 y = acc[i][ct];
                        if (col < L)
                            gst((u32x2*)(o + col), u32x2{pack_bf16(y[0] * inv, y[1] * inv), pack_bf16(y[2] * inv, y[3] * inv)});
                    }
                } else {
                    float* o = p.part + ((size_t)slot * ROWS + lr) * (128u * LC);
#pragma unroll
                    for (uint32_t ct = 0; ct < CT; ct++) gst((f32x4*)(o + 32u * LC * wv + 16u * ct + 4u * g), acc[i][ct]);
                    if (wv == 0 && g == 0) {
                        p.part_ml[2u * (slot * ROWS + lr)] = m[i];
                        p.part_ml[2u * (slot * ROWS + lr) + 1u] = sum;
                    }
                }
            }
        }
        if (!whole && tid == (kt0 == 0 ? 1u : 0u)) {  // the thread that cleared it
            const uint64_t start = base + (uint64_t)rt * q.nkt;
            uint32_t* desc = p.desc + 4 * slot;
            desc[0] = r + 1u;
            desc[1] = rt;
            desc[2] = (uint32_t)(start / f.per);
            desc[3] = (uint32_t)((start + q.nkt - 1) / f.per);
        }
        __syncthreads();
        if (tid == 0) bad_page = 0u;
        __syncthreads();
    }
}

// Joins the parts of split row tiles: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s
// - M) l_s. Each work-group that a tile's keys were spread over joins its share
// of the tile's rows, so the parts are read by as many work-groups as wrote
// them. Work-group (c, k): slot 2 c + k's tile. A row's parts are summed by the
// four waves in turn (wave w parts w, w + 4, ...), lane the columns 4 lane + 256 j,
// and the four sums in order.
template <int ROWS, int LC, bool OBF>
__global__ __launch_bounds__(256) void tree_join_kernel(Tree p) {
    constexpr uint32_t COLS = 128 * LC, NV = (COLS + 255) / 256;
    __shared__ f32x4 sums[4][NV][64];
    __shared__ float wsum[4];
    const uint32_t c = blockIdx.x, lane = threadIdx.x & 63u, wv = uni(threadIdx.x >> 6);
    const uint32_t* desc = p.desc + 4 * (2 * c + blockIdx.y);
    if (desc[0] == 0) return;
    uint32_t status = 0;
    const Req q = request<ROWS>(p, desc[0] - 1u, status);
    const uint32_t rt = desc[1], c0 = desc[2], S = desc[3] - c0 + 1u, H = p.a.n_heads, L = p.a.cache.kv_lora_rank;
    const uint32_t all = q.nodes * H - rt * ROWS, rows = all < ROWS ? all : ROWS;
    for (uint32_t lr = rows * (c - c0) / S; lr < rows * (c - c0 + 1u) / S; lr++) {
        // part s: slot 2 c0 + 1 for s = 0, else 2 (c0 + s)
        auto at = [&](uint32_t s) { return (size_t)(s == 0 ? 2u * c0 + 1u : 2u * (c0 + s)) * ROWS + lr; };
        float M = kNone;
        for (uint32_t s = lane; s < S; s += 64) M = fmaxf(M, p.part_ml[2 * at(s)]);
        for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        f32x4 y[NV];
#pragma unroll
        for (uint32_t k = 0; k < NV; k++) y[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll 4
        for (uint32_t s = wv; s < S; s += 4) {
            const float* ml = p.part_ml + 2 * at(s);
            const float w = exp2_(ml[0] - M);
            sum += w * ml[1];
            const float* o = p.part + at(s) * COLS + 4u * lane;
#pragma unroll
            for (uint32_t k = 0; k < NV; k++) {
                if (4u * lane + 256u * k < COLS) {
                    const f32x4 v = gld((const f32x4*)(o + 256u * k));
#pragma unroll
                    for (int j = 0; j < 4; j++) y[k][j] += w * v[j];
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < NV; k++) sums[wv][k][lane] = y[k];
        if (lane == 0) wsum[wv] = sum;
        __syncthreads();
        if (wv < NV) {
            const float total = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
            const float inv = total == 0.f ? 0.f : 1.0f / total;
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++)
                v[j] = ((sums[0][wv][lane][j] + sums[1][wv][lane][j]) + (sums[2][wv][lane][j] + sums[3][wv][lane][j])) * inv;
            const uint32_t row = rt * ROWS + lr, node = row / H, h = row - node * H, col = 4u * lane + 256u * wv;
            const size_t o = (size_t)(q.t0 + node) * p.a.out_stride + (size_t)h * L + col;
            if (col < L) {
                if (OBF) gst((u32x2*)((uint16_t*)p.a.d_out + o), u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])});
                else gst((f32x4*)((float*)p.a.d_out + o), v);
            }
        }
        __syncthreads();
    }
}
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

uint32_t lat_class(const wl_tree_attn& a) {  // 128-column blocks of a row's latent part, as the kernels have them
    const uint32_t b = (a.cache.kv_lora_rank + 127) / 128;
    return b <= 1 ? 1 : b <= 2 ? 2 : 4;
}
uint32_t row_class(const wl_tree_attn& a) {  // rows of a work-group's block
    const uint64_t rows = (uint64_t)a.n_heads * (a.n_req ? (a.n_tokens + a.n_req - 1) / a.n_req : 1);
    return rows > 32 ? 64 : rows > 16 ? 32 : 16;
}

size_t tree_scratch(const wl_tree_attn& a) {
    const size_t rows = 2 * kGrid * 64;
    return rows * (128 * lat_class(a) + 2) * 4 + 2 * kGrid * 16;
}

template <int MT, int RG, int LC>
int run_bf16(const Tree& p, hipStream_t st) {
    constexpr int ROWS = 16 * MT * RG;
    hipLaunchKernelGGL((tree_bf16_kernel<MT, RG, LC>), dim3(kGrid), dim3(256 * RG), 0, st, p, 1u);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL((tree_join_kernel<ROWS, LC, true>), dim3(kGrid, 2), dim3(256), 0, st, p);
    return (int)hipGetLastError();
}

int launch_tree(const wl_tree_attn& a, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    Tree p{};
    p.a = a;
    p.psh = 31u - (uint32_t)__builtin_clz(a.cache.page_size);
    p.scale2 = a.scale * 1.44269504088896340736f;
    const uint32_t lc = lat_class(a), rows = row_class(a);
    p.part = (float*)a.d_scratch;
    p.part_ml = p.part + (size_t)2 * kGrid * 64 * 128 * lc;
    p.desc = (uint32_t*)(p.part_ml + (size_t)2 * kGrid * 64 * 2);
    if (a.dtype == WL_TYPE_BF16) {
        if (rows == 64) return lc == 4 ? run_bf16<2, 2, 4>(p, st) : lc == 2 ? run_bf16<2, 2, 2>(p, st) : run_bf16<2, 2, 1>(p, st);
        if (rows == 32) return lc == 4 ? run_bf16<1, 2, 4>(p, st) : lc == 2 ? run_bf16<1, 2, 2>(p, st) : run_bf16<1, 2, 1>(p, st);
        return lc == 4 ? run_bf16<1, 1, 4>(p, st) : lc == 2 ? run_bf16<1, 1, 2>(p, st) : run_bf16<1, 1, 1>(p, st);
    }
    const dim3 g(a.n_req, (a.n_heads + 3) / 4, 8);
    if (a.cache.dtype == WL_TYPE_BF16) hipLaunchKernelGGL((tree_attn_kernel<false, true>), g, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((tree_attn_kernel<false, false>), g, dim3(256), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace paged
}  // namespace wl
