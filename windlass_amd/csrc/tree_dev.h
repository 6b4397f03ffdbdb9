// tree_dev.h — what the kernels of attention over the paged cache share
// (tree_attn.hip, tree_mx4.hip): the work's split, a walk's place in it, parts of
// row tiles, and where LDS rows lie. Not public ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "paged.h"
#include "paged_dev.h"
#include "window.h"

namespace wl {
namespace paged {
namespace {

constexpr uint32_t kKT = 32;    // keys of a tile
// Key tiles of a walk at least: a shorter one's parts cost more to join than it saves.
// Both launches in us at 1, 2, 3 and 4: one token x 64 heads over 4096 keys 31.0, 27.5, 27.8,
// 28.0, with 32-bit queries 30.4, 28.6, 29.9, 31.6, 32 bits throughout (two of 16 keys)
// 35.5, 38.4, 42.9, 49.8; 12 requests of up to 5 nodes, 32-bit queries, 22.1, 22.1, 22.9, 24.9.
constexpr uint32_t kMinPer = 2;
constexpr uint32_t kGrid = 256;      // work-groups of a launch of the 16-bit kernel: one per CU (LDS and registers allow one)
constexpr uint32_t kGridF32 = 512;   // of the 32-bit one: two per CU
constexpr uint32_t kRows16 = 64, kRows32 = 32;  // rows of their tiles
constexpr float kNone = -3.0e38f;  // the running maximum of a row that has seen no key


typedef __attribute__((ext_vector_type(4))) short s16x4;
#define WL_LDS(p) ((__attribute__((address_space(3))) void*)(p))

constexpr uint32_t kDesc = 16;
// What a launch needs beside the call's arguments.
struct Tree {
    wl_tree_attn a;
    uint32_t psh;      // log2 page_size
    float scale2;      // scale * log2(e): scores in powers of two
    float* part;       // [2 grid][rows][cols] unnormalised sums of split tiles
    float* part_ml;    // [2 grid][rows][2] their maxima and weight sums
    uint32_t* desc;    // [2 grid][kDesc] the parts' row tiles, as name_part writes them, or 0
    uint32_t window, sinks;  // of a windowed call (the kernels' WIN)
};

// ---- the work and its split --------------------------------------------------
// A request's rows (node, head) come in tiles of ROWS, its keys in tiles of
// kKT; a unit is one of each. The units of all requests stand in one row, and
// work-group c takes [c per, c per + per) of them, so every work-group has the
// same number of key tiles to go through, whatever the requests' lengths. A
// request's keys are cut into chunks of at least `per` tiles (one chunk, if they
// are fewer); its units come chunk by chunk, in a chunk row tile by row tile:
// the row tiles that run at the same time are at the same keys, which the L2 of
// their XCD then holds once for all of them. (Work-group b runs on XCD b % 8:
// c = (b % 8)(G / 8) + b / 8.) A row tile's units count from its keys' end: the next
// work-group, which has the rest of a row tile that this one ends with, then begins at
// the chunk's first key as this one did, and not some tiles ahead (64 requests of 8 nodes,
// 16-bit rows: 207 us and 198; through a window 149 and 142, 717 MB fetched and 298; 32-bit
// queries over these rows 385 and 370, over 32-bit ones 360 and 349, 3 of 64 nodes 614 and 589).
// A row tile that one work-group has whole is finished there; the others leave their
// parts in the scratch for the second launch, at most two per work-group: its first
// walk's and its last one's.
// Where there are fewer row tiles than work-groups that is mostly two walks each, and
// a walk's start, its end and its part cost as much as some kSlack tiles. So where
// pieces of row tiles (all of a request's equally long, as many as need be) at most
// that much longer than `per` (and a sixteenth) are no more than the work-groups,
// work-group c takes piece c. (Requests without tokens change nothing of this, as
// long as a launch has a thread for each: up to 256, 512 in work-groups of eight waves.)
// One request of 64 nodes over 8192 keys, 32 bits: 222 us
// without, 207 with; 5 of 7 nodes 67 and 59; 12 of 5 nodes 28 and 23; 32 contexts 191 and 179. Requests of
// one row tile, 16-bit queries: 32 contexts of up to 65536 keys 180 and 170, of 4-bit rows 129 and 121, these
// through a window of 4096 57 and 46; 8 of up to 3016 keys 25 and 19; with 32-bit queries 5 of 16 heads over
// up to 9000 keys 34 and 29, 100 of up to 9000 and one of 4096 as without. (They need no chunks: their keys stand
// in a row; of one such request alone that makes equal pieces by itself.)
constexpr uint32_t kSlack = 6;
//
// Through a window (WIN) a request's keys are those that some node may see: tiles
// [0, st) with the sinks and those from the first key on that its first node sees;
// `skip` tiles between them are no units. A walk counts the others (nkt); the first
// key of its tile t is key_of(t). Nodes of a request see windows a few keys apart, so
// only the tiles at the sinks' end, at the window's beginning and with nodes are masked.
// 32 single tokens through a window of 4096 with 4 sinks, 4-bit rows: 46 us (all keys 121);
// 64 requests of up to 8 nodes through 2048 with 64 sinks, 16-bit rows: 142 us.
struct Req {
    uint32_t t0, nodes, len, keys, nrt, nkt, flaw;  // flaw: WL_PAGED_E_* (its rows get NaN)
    uint32_t st, skip;
};
template <bool WIN>
WL_DEV uint32_t key_of(const Req& q, uint32_t t) {
    return (WIN && t >= q.st ? t + q.skip : t) * kKT;
}
// Whether keys [k0, k0 + n) have to be masked: nodes are among them (or keys behind the
// last one), or keys that a window passes over for some node.
template <bool WIN>
WL_DEV bool is_masked(const Tree& p, const Req& q, uint32_t k0, uint32_t n) {
    return k0 + n > q.len || (WIN && window_masks(q.len, q.nodes, p.window, p.sinks, k0, n));
}
// What node nd of a request sees: of the nodes those in the result (a bit each), of
// the keys before them those from `low` on and the sinks. Its position is the number
// of its ancestors behind len, an ancestor's the number of those before it.
template <bool WIN>
WL_DEV uint64_t sees(const Tree& p, const Req& q, uint32_t nd, uint32_t& low) {
    uint64_t bits = p.a.d_mask ? p.a.d_mask[q.t0 + nd] : (2ull << nd) - 1ull;
    low = 0;
    if (WIN) {
        const uint64_t below = bits & ((1ull << nd) - 1ull);
        const uint32_t depth = (uint32_t)__popcll(below);
        low = window_from(q.len + depth, p.window);
        const uint32_t drop = depth >= p.window ? depth - p.window + 1u : 0u, sunk = p.sinks > q.len ? p.sinks - q.len : 0u;
        uint64_t left = below;
        for (uint32_t i = 0; i < drop; i++) {  // at most 63
            const uint64_t bit = left & (0ull - left);
            left ^= bit;
            if (i >= sunk) bits ^= bit;
        }
    }
    return bits;
}
template <uint32_t ROWS, bool WIN>
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
    q.st = ~0u;
    if (WIN && !q.flaw) {
        const Skip skip = window_skip(q.len, p.window, p.sinks, kKT);
        q.st = skip.at;
        q.skip = skip.n;
        q.nkt -= skip.n;
    }
    return q;
}

// a / b, in 32 bits where both fit (64-bit quotients take some hundred instructions).
WL_DEV uint64_t div64(uint64_t a, uint64_t b) {
    return ((a | b) >> 32) == 0 ? (uint64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// The sum of x over this lane and those below it: within rows of 16 lanes, then the
// rows' last lanes handed on. (Shuffles go through LDS, some 130 clocks a step.)
template <int CTRL, int ROWMASK>
WL_DEV uint32_t dpp0(uint32_t x) {  // lanes without a source get 0
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWMASK, 0xf, false);
}
template <int CTRL, int ROWMASK>
WL_DEV uint64_t dpp0(uint64_t x) {
    return (uint64_t)dpp0<CTRL, ROWMASK>((uint32_t)(x >> 32)) << 32 | dpp0<CTRL, ROWMASK>((uint32_t)x);
}
template <class T>
WL_DEV T sum_up(T x) {
    x += dpp0<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
    x += dpp0<0x112, 0xf>(x);
    x += dpp0<0x114, 0xf>(x);
    x += dpp0<0x118, 0xf>(x);
    x += dpp0<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    x += dpp0<0x143, 0xc>(x);
    return x;
}

// The launch's units (or pieces), and the request (with its first one) that unit
// u0 = c per (piece c) falls into. Each thread sums the requests of its share; tmp: two
// words per wave, and ten; rq: a pair per thread.
WL_DEV uint64_t uni64(uint64_t x) { return (uint64_t)uni((uint32_t)(x >> 32)) << 32 | uni((uint32_t)x); }
struct Place {
    uint64_t total, per, u0, base;
    uint32_t r, pieces;
    Req q;
};
constexpr uint32_t kTries = 8;
template <uint32_t ROWS, uint32_t THREADS, uint32_t GRID, bool WIN>
WL_DEV Place find_place(const Tree& p, uint32_t c, uint32_t min_per, uint64_t* tmp, u32x2* rq, Req* found) {
    constexpr uint32_t NW = THREADS / 64;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6, R = p.a.n_req;
    const uint32_t share = (R + THREADS - 1u) / THREADS;
    uint64_t mine = 0;
    uint32_t status = 0, tiles = 0;
    Req q{};
    for (uint32_t i = 0; i < share; i++) {
        const uint32_t r = tid * share + i;
        if (r < R) {
            q = request<ROWS, WIN>(p, r, status);
            mine += (uint64_t)q.nrt * q.nkt;
            tiles += q.nrt < GRID ? q.nrt : GRID;  // (of a refused request it may be any number)
        }
    }
    rq[tid] = u32x2{q.nrt, q.nkt};
    if (c == 0 && status) set_status(p.a.d_status, status);
    const uint64_t inc = sum_up(mine);
    tiles = sum_up(tiles);
    if (lane == 63) {
        tmp[wv] = inc;
        tmp[NW + 2 + wv] = tiles;
    }
    __syncthreads();
    Place f;
    f.total = 0;
    uint64_t all = 0;
#pragma unroll
    for (uint32_t w = 0; w < NW; w++) {
        f.total += tmp[w];
        all += tmp[NW + 2 + w];
    }
    f.per = (f.total + GRID - 1) / GRID;
    if (f.per < min_per) f.per = min_per;
    f.u0 = (uint64_t)c * f.per;
    f.pieces = 0;
    uint64_t at = inc - mine;
    for (uint32_t w = 0; w < wv; w++) at += tmp[w];
    if (share == 1 && (R > 1 || rq[0][0] > 1) && all < GRID && (f.total >> 32) == 0) {
        // the least of some lengths with which the pieces are no more than the work-groups
        const uint32_t per = (uint32_t)f.per, step = (kSlack + per / 16u + kTries - 2u) / (kTries - 1u);
        for (uint32_t k = wv; k < kTries; k += NW) {
            const uint32_t len = per + k * step;
            uint32_t n = 0;
            for (uint32_t r = lane; r < R; r += 64) n += rq[r][0] * ((rq[r][1] + len - 1u) / len);
            n = sum_up(n);
            if (lane == 63) ((uint32_t*)(tmp + 2 * NW + 2))[k] = n;
        }
        __syncthreads();
        for (uint32_t k = kTries; k-- > 0;)
            if (((const uint32_t*)(tmp + 2 * NW + 2))[k] <= GRID) f.pieces = per + k * step;
        f.pieces = uni(f.pieces);
    }
    if (f.pieces) {
        f.per = f.pieces;
        f.u0 = c;
        mine = q.nrt * ((q.nkt + f.pieces - 1u) / f.pieces);
        const uint32_t sum = sum_up((uint32_t)mine);
        if (lane == 63) tmp[wv] = sum;
        __syncthreads();
        f.total = 0;
        at = sum - mine;
#pragma unroll
        for (uint32_t w = 0; w < NW; w++) {
            if (w < wv) at += tmp[w];
            f.total += tmp[w];
        }
    }
    if (f.u0 >= at && f.u0 < at + mine) {  // one thread at most
        uint32_t r = tid * share;
        if (share > 1) {
            for (;; r++) {
                q = request<ROWS, WIN>(p, r, status);
                const uint64_t n = (uint64_t)q.nrt * q.nkt;
                if (f.u0 < at + n) break;
                at += n;
            }
        }
        tmp[NW] = at;
        tmp[NW + 1] = r;
        *found = q;
    }
    __syncthreads();
    f.total = uni64(f.total);
    f.per = uni64(f.per);
    f.base = uni64(tmp[NW]);
    f.r = uni((uint32_t)tmp[NW + 1]);
    f.q = Req{uni(found->t0),  uni(found->nodes), uni(found->len), uni(found->keys),
              uni(found->nrt), uni(found->nkt),   uni(found->flaw), ~0u, 0u};
    if (WIN) {
        f.q.st = uni(found->st);
        f.q.skip = uni(found->skip);
    }
    return f;
}

// Chunk j of a request's nc: key tiles [chunk_at(j), chunk_at(j + 1)), each at least `per` if nc > 1.
WL_DEV uint32_t chunks(const Req& q, uint64_t per) { return q.nrt == 1 || per > q.nkt ? 1u : q.nkt / (uint32_t)per; }
WL_DEV uint32_t pieces_of(const Req& q, uint32_t len) { return (q.nkt + len - 1u) / len; }
WL_DEV uint32_t chunk_at(const Req& q, uint32_t nc, uint32_t j) { return (uint32_t)div64((uint64_t)j * q.nkt, nc); }

WL_DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
WL_DEV bool has_nonfinite(u32x4 v) {
    bool f = false;
#pragma unroll
    for (int i = 0; i < 4; i++)
        f |= (v[i] & 0x7F80u) == 0x7F80u || (v[i] & 0x7F800000u) == 0x7F800000u;
    return f;
}
// The walks of work-group c: a row tile's keys, or a part of them.
struct Walk {
    Req q;
    uint64_t base;
    uint32_t r, rt, kt0, kt1, slot;
};
template <uint32_t ROWS, bool WIN>
struct Walks {
    const Tree& p;
    const Place f;
    const uint64_t u1;
    const uint32_t c;
    uint64_t u;
    uint32_t status;
    Walk next;
    __device__ __forceinline__ Walks(const Tree& t, const Place& pl, uint32_t wg)
        : p(t), f(pl), u1(end(pl)), c(wg), u(pl.u0), status(0), next{pl.q, pl.base, pl.r, 0, 0, 0, 0} {}
    static __device__ __forceinline__ uint64_t end(const Place& pl) {
        const uint64_t u = pl.u0 + (pl.pieces ? 1u : pl.per);
        return u < pl.total ? u : pl.total;  // (a work-group without work begins behind it)
    }
    __device__ __forceinline__ bool more() const { return u < u1; }
    __device__ __forceinline__ void find() {  // the walk that begins at unit u < u1, from the last one's request on
        Walk& w = next;
        if (f.pieces) {
            const uint32_t i = (uint32_t)(u++ - w.base), nc = uni(pieces_of(w.q, f.pieces)), j = uni(i / w.q.nrt);
            const uint32_t len = uni(w.q.nkt / nc), longer = w.q.nkt - len * nc;  // the first ones one tile more
            w.rt = uni(i - j * w.q.nrt);
            w.kt0 = uni(j * len + (j < longer ? j : longer));
            w.kt1 = uni(w.kt0 + len + (j < longer ? 1u : 0u));
            w.slot = 2u * c;
            return;
        }
        while (u >= w.base + (uint64_t)w.q.nrt * w.q.nkt) {  // the next request that has units
            w.base += (uint64_t)w.q.nrt * w.q.nkt;
            w.q = request<ROWS, WIN>(p, ++w.r, status);
        }
        const uint64_t o = u - w.base;
        const uint32_t nc = uni(chunks(w.q, f.per)), j = uni((uint32_t)div64((div64(o, w.q.nrt) + 1) * nc - 1, w.q.nkt));
        const uint32_t ka = uni(chunk_at(w.q, nc, j)), kb = uni(chunk_at(w.q, nc, j + 1));
        const uint64_t oj = o - (uint64_t)w.q.nrt * ka;
        w.rt = uni((uint32_t)div64(oj, kb - ka));
        const uint32_t k0 = (uint32_t)(oj - (uint64_t)w.rt * (kb - ka)), left = kb - ka - k0, n = uni(u1 - u < left ? (uint32_t)(u1 - u) : left);
        w.kt1 = uni(kb - k0);  // (from the chunk's end)
        w.kt0 = w.kt1 - n;
        w.slot = 2u * c + (u == f.u0 ? 0u : 1u);
        u += n;
    }
    __device__ __forceinline__ uint32_t rows(const Walk& w) const {
        const uint32_t n = w.q.nodes * p.a.n_heads - w.rt * ROWS;
        return n < ROWS ? n : ROWS;
    }
    // The page of DR consecutive keys of tile t, from its key k0 on (pages have at
    // least 8 rows, and DR is at most 8); behind the last key, the last key's
    __device__ __forceinline__ int32_t page(const Walk& w, uint32_t t, uint32_t k0) const {
        const uint32_t key = key_of<WIN>(w.q, t) + k0;
        return p.a.d_table[(size_t)w.r * p.a.max_pages + ((key < w.q.keys ? key : w.q.keys - 1u) >> p.psh)];
    }
    // names the row tile of the walk's part for the second launch
    __device__ __forceinline__ void name_part(const Walk& w) const {
        uint32_t* desc = p.desc + kDesc * w.slot;
        desc[0] = 1u;
        desc[1] = w.rt;
        *(uint64_t*)(desc + 2) = w.base;
        *(uint64_t*)(desc + 4) = f.per;
        desc[6] = f.pieces;
        desc[7] = w.q.t0;
        desc[8] = w.q.nodes;
        desc[9] = w.q.nrt;
        desc[10] = w.q.nkt;
    }
};
// One lane's share of a row of sums (4 columns of every 16 from column `col` on,
// n16 of them): finished, or as a part.
template <uint32_t ROWS, int LC, bool OBF, uint32_t N16>
WL_DEV void put_row(const Tree& p, const Walk& w, bool whole, uint32_t lr, float sum, const f32x4* y, uint32_t col) {
    if (whole) {
        const uint32_t H = p.a.n_heads, L = p.a.cache.kv_lora_rank;
        const uint32_t row = w.rt * ROWS + lr, node = row / H, h = row - node * H;
        const size_t o = (size_t)(w.q.t0 + node) * p.a.out_stride + (size_t)h * L + col;
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
        for (uint32_t k = 0; k < N16; k++) {
            if (col + 16u * k >= L) continue;
            const f32x4 v = {y[k][0] * inv, y[k][1] * inv, y[k][2] * inv, y[k][3] * inv};
            if (OBF) gst((u32x2*)((uint16_t*)p.a.d_out + o + 16u * k), u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])});
            else gst((f32x4*)((float*)p.a.d_out + o + 16u * k), v);
        }
    } else {
        float* o = p.part + ((size_t)w.slot * ROWS + lr) * (128u * LC) + col;
#pragma unroll
        for (uint32_t k = 0; k < N16; k++) gst((f32x4*)(o + 16u * k), y[k]);
    }
}

// s_waitcnt vmcnt(N): all but the last N memory operations of this wave are done.
template <uint32_t N>
WL_DEV void vm_wait() {
    static_assert(N < 64u, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt((N & 15u) | ((N >> 4) << 14) | 0x0F70u);
}
// A barrier that orders LDS accesses of the waves' instructions only: DMA into
// LDS, loads and stores go on across it (a release fence would wait for them).
WL_DEV void ring_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// x, of which nothing is computed ahead of this place: what is derived from it holds
// no register before, over all the rest of the kernel.
WL_DEV uint32_t afresh(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// LDS serves a 16-byte read 16 lanes at a time, lanes 0-3, 12-15, 20-27 and 4-11,
// 16-19, 28-31 of either half wave: for an MFMA operand (lane = row + 16 x chunk)
// those are 8 rows at an even chunk and the other 8 at the odd one beside it. Key
// rows lie 32 bytes more than a multiple of 256 apart, which puts these 16 into 16
// different places of the 256 bytes that the banks cover, as it does the 8 rows x 2
// chunks that half a wave reads transposed. Rows of 128 and 64 bytes (rotary parts,
// weights) have their chunk c at c ^ swz8(row) and c ^ swz4(row) instead.
// Measured: 236 bytes a clock and CU (32 without).
constexpr uint32_t kPad = 32;
WL_DEV constexpr uint32_t swz8(uint32_t row) { return (row & 2u) | ((row & 8u) >> 1); }
WL_DEV constexpr uint32_t swz4(uint32_t row) { return (row & 8u) >> 2; }

constexpr float kMost = 0x1p64f;  // 2^31 such weights sum to 2^95
// How far above its true maximum the reference of a walk that is done again lies, in
// powers of two: the weights of all its keys then sum to 1/2 at the most, and no sum of
// them and values is more than the largest of these. (The exponentials' arguments are
// rounded at that size, 2^-20 for up to 2^15 keys. Scores of such a walk, 64 powers of
// two apart, have no finer step; where only values are large, it is what they cost.)
WL_DEV float lift_of(uint32_t keys) { return (float)(33u - (uint32_t)__clz((int)(keys - 1u))); }  // 1 + ceil(log2 keys), keys >= 2
// Whether a value is not finite (a NaN is the largest of any).
template <uint32_t N>
WL_DEV bool nonfinite(const f32x4 (&y)[N]) {
    float z = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < N; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) z = __builtin_elementwise_maximum(z, fabsf(y[k][j]));
    return !(z <= 3.402823466e38f);
}

// Joins the parts of split row tiles: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s
// - M) l_s. Each part's writer (slot blockIdx.x) has Z work-groups here that
// join its share of the tile's rows, so the parts are read by as many CUs as
// wrote them. The tile's parts are listed first, a thread per chunk of its keys.
// Of few parts a wave joins a row by itself; many are dealt out to the four
// waves, a quarter each, and their sums added in order. Lane: columns 4 lane + 256 k.
// Parts to read and their number bound it: 33 MB in 12 us for 512 parts of 32 rows,
// 6.7 us for one token's 65.
constexpr uint32_t kManyParts = 16;
// The parts' weights are 1 at the most: as many finite sums, each times this, are finite.
constexpr float kPart = 0.5f / (2 * kGridF32);
template <uint32_t GRID, uint32_t ROWS, int LC, bool OBF>
__global__ __launch_bounds__(256) void tree_join_kernel(Tree p) {
    constexpr uint32_t COLS = 128 * LC, NV = (COLS + 255) / 256, Z = 1024 / GRID;
    __shared__ f32x4 sums[4][NV][64];
    __shared__ float weight[4][2 * GRID];
    __shared__ uint32_t count[4], list[2 * GRID];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = uni(tid >> 6), mine = blockIdx.x;
    const uint32_t* desc = p.desc + kDesc * mine;
    if (desc[0] == 0) return;
    Req q{};  // as the first launch found it, in one read
    q.t0 = desc[7], q.nodes = desc[8], q.nrt = desc[9], q.nkt = desc[10];
    const uint32_t rt = desc[1], H = p.a.n_heads, L = p.a.cache.kv_lora_rank;
    const uint64_t base = *(const uint64_t*)(desc + 2), per = *(const uint64_t*)(desc + 4);
    const uint32_t pieces = desc[6];
    uint32_t S;
    if (pieces) {
        S = pieces_of(q, pieces);
        for (uint32_t i = tid; i < S; i += 256) list[i] = 2u * ((uint32_t)base + i * q.nrt + rt);
        __syncthreads();
    } else if (chunks(q, per) == 1) {
        const uint64_t start = base + (uint64_t)rt * q.nkt;
        const uint32_t w0 = (uint32_t)div64(start, per);
        S = (uint32_t)div64(start + q.nkt - 1, per) - w0 + 1u;
        for (uint32_t i = tid; i < S; i += 256) list[i] = 2u * (w0 + i) + (start <= (w0 + i) * per ? 0u : 1u);
        __syncthreads();
    } else {
        constexpr uint32_t C = GRID / 256;  // chunks of a thread
        const uint32_t nc = chunks(q, per);
        uint64_t start[C];
        uint32_t w0[C], nw[C], all = 0;
#pragma unroll
        for (uint32_t i = 0; i < C; i++) {
            const uint32_t ch = C * tid + i;
            start[i] = 0;
            w0[i] = nw[i] = 0;
            if (ch < nc) {
                const uint32_t ka = chunk_at(q, nc, ch), kb = chunk_at(q, nc, ch + 1);
                start[i] = base + (uint64_t)q.nrt * ka + (uint64_t)rt * (kb - ka);
                w0[i] = (uint32_t)div64(start[i], per);
                nw[i] = (uint32_t)div64(start[i] + (kb - ka) - 1, per) - w0[i] + 1u;
            }
            all += nw[i];
        }
        uint32_t inc = all;
        for (uint32_t o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(inc, o, 64);
            if (lane >= o) inc += v;
        }
        if (lane == 63) count[wv] = inc;
        __syncthreads();
        uint32_t at = inc - all;
        for (uint32_t w = 0; w < wv; w++) at += count[w];
#pragma unroll
        for (uint32_t i = 0; i < C; i++)
            for (uint32_t k = 0; k < nw[i]; k++)  // a work-group's first walk has its even slot
                list[at++] = 2u * (w0[i] + k) + (start[i] <= (w0[i] + k) * per ? 0u : 1u);
        __syncthreads();
        S = count[0] + count[1] + count[2] + count[3];
    }
    uint32_t idx = 0;
    for (uint32_t s = lane; s < S; s += 64)
        if (list[s] == mine) idx = s + 1u;
    for (int o = 32; o > 0; o >>= 1) idx |= __shfl_xor(idx, o, 64);
    idx = uni(idx) - 1u;
    const uint32_t all = q.nodes * H - rt * ROWS, rows = all < ROWS ? all : ROWS;
    const bool many = S >= kManyParts;
    const uint32_t r0 = rows * idx / S, r1 = rows * (idx + 1u) / S;
    for (uint32_t lr = r0 + (many ? blockIdx.y : 4u * blockIdx.y + wv); lr < r1; lr += many ? Z : 4u * Z) {
        auto at = [&](uint32_t s) { return (size_t)list[s] * ROWS + lr; };
        f32x4 y[NV];
#pragma unroll
        for (uint32_t k = 0; k < NV; k++) y[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
        auto take = [&](uint32_t s, float w) {
            const float* o = p.part + at(s) * COLS + 4u * lane;
#pragma unroll
            for (uint32_t k = 0; k < NV; k++) {
                if (COLS % 256 == 0 || 4u * lane < COLS) {
                    const f32x4 v = gld((const f32x4*)(o + 256u * k));
#pragma unroll
                    for (int j = 0; j < 4; j++) y[k][j] += w * v[j];
                }
            }
        };
        float M = kNone;
        for (uint32_t s = lane; s < S; s += 64) M = fmaxf(M, p.part_ml[2 * at(s)]);
        for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        if (!many) {
#pragma unroll 4
            for (uint32_t s = 0; s < S; s++) {
                const float* ml = p.part_ml + 2 * at(s);
                const float w = exp2_(ml[0] - M) * kPart;
                sum += w * ml[1];
                take(s, w);
            }
        } else {
            for (uint32_t s = lane; s < S; s += 64) {
                const float w = exp2_(p.part_ml[2 * at(s)] - M) * kPart;
                weight[wv][s] = w;
                sum += w * p.part_ml[2 * at(s) + 1];
            }
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
            const uint32_t s1 = S * (wv + 1u) / 4u;
#pragma unroll 4
            for (uint32_t s = S * wv / 4u; s < s1; s++) take(s, weight[wv][s]);
        }
        const uint32_t row = rt * ROWS + lr, node = row / H, h = row - node * H;
        const size_t out = (size_t)(q.t0 + node) * p.a.out_stride + (size_t)h * L;
        auto put = [&](f32x4 v, float total, uint32_t k) {
            const float inv = total == 0.f ? 0.f : 1.0f / total;
            const uint32_t col = 4u * lane + 256u * k;
            if (col < L) {
                if (OBF)
                    gst((u32x2*)((uint16_t*)p.a.d_out + out + col),
                        u32x2{pack_bf16(v[0] * inv, v[1] * inv), pack_bf16(v[2] * inv, v[3] * inv)});
                else
                    gst((f32x4*)((float*)p.a.d_out + out + col), f32x4{v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv});
            }
        };
        if (!many) {
#pragma unroll
            for (uint32_t k = 0; k < NV; k++) put(y[k], sum, k);
            continue;
        }
#pragma unroll
        for (uint32_t k = 0; k < NV; k++) sums[wv][k][lane] = y[k];
        __syncthreads();
        if (wv < NV) {
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++)
                v[j] = (sums[0][wv][lane][j] + sums[1][wv][lane][j]) + (sums[2][wv][lane][j] + sums[3][wv][lane][j]);
            put(v, sum, wv);
        }
        __syncthreads();
    }
}

inline uint32_t lat_class(const wl_tree_attn& a) {  // 128-column blocks of a row's latent part, as the kernels have them
    const uint32_t b = (a.cache.kv_lora_rank + 127) / 128;
    return b <= 1 ? 1 : b <= 2 ? 2 : 4;
}
inline size_t part_rows(const wl_tree_attn& a) { return a.dtype == WL_TYPE_BF16 ? 2 * kGrid * kRows16 : 2 * kGridF32 * kRows32; }

// run(LC) of the call's class.
template <class F>
int by_class(const wl_tree_attn& a, F run) {
    const uint32_t lc = lat_class(a);
    return lc == 4 ? run(std::integral_constant<int, 4>{}) : lc == 2 ? run(std::integral_constant<int, 2>{})
                                                                     : run(std::integral_constant<int, 1>{});
}
inline Tree make_tree(const wl_tree_attn& a, uint32_t window, uint32_t sinks) {
    Tree p{};
    p.a = a;
    p.psh = 31u - (uint32_t)__builtin_clz(a.cache.page_size);
    p.scale2 = a.scale * 1.44269504088896340736f;
    p.part = (float*)a.d_scratch;
    p.part_ml = p.part + part_rows(a) * 128 * lat_class(a);
    p.desc = (uint32_t*)(p.part_ml + part_rows(a) * 2);
    p.window = window;
    p.sinks = sinks;
    return p;
}
}  // namespace
}  // namespace paged
}  // namespace wl
