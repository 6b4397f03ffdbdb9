// tree_attn.hip — attention of trees of drafted tokens over a paged cache of
// latent rows (wl_paged_tree_attention, wl_paged_window_attention); 16-bit queries
// over 4-bit rows are tree_mx4.hip's.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "tree_dev.h"

namespace wl {
namespace paged {
namespace {

// ---- 16-bit queries and cache --------------------------------------------------
// 64 rows (node, head) against 32 keys at a time, two groups of four waves with 32
// rows each. (One group for requests of at most 32 rows: one token of 32 heads over up to
// 65536 keys, 32 requests, 512 columns, 163 us against 165; 256 columns 137 against 130,
// 128 columns and 16 heads 121 against 113.) In a group
//   S^T[keys][rows] = K Q^T: wave w takes row tile w / 2 and 16-key tile w % 2;
//           its 16 rows' queries stay in its registers through the whole walk
//           (4 LC + 2 steps of 32 columns);
//   P = 2^(S - m) in bf16, through LDS, to the group's waves;
//   O^T[cols][rows] += V^T P^T: wave w has columns [32 LC w, + 32 LC); the key
//           rows are read again, transposed (ds_read_b64_tr_b16).
// One barrier a tile: between two of them a wave makes the scores of tile t, then
// sums tile t - 1 with the exponentials of tile t between the products.
// m is a reference, not the maximum: that of the walk's first tile. Weights may
// exceed 1 and lose nothing by it (bf16 and f32 keep their relative precision); only
// where a weight passes kMost, or a sum of weighted values is not finite, the walk is
// done again, after one over the scores alone for the true maxima, with a reference
// above them (lift_of). So nothing is rescaled, and finite rows have finite results.
// Key rows come into a ring of four tiles in LDS by DMA (16 bytes a lane): rows
// behind the last key and columns behind the row's are read as zeros by the
// resource's bounds. While tiles t - 1 and t are worked on, tile t + 2 is called
// for between products; before the barrier each wave waits for its rows of t + 1.
// P in bf16: a weight p is off by 2^-8 of itself at the most, and the sum that it is
// divided by is of the rounded weights. So a result stays a mean of the values c: it is
// off by 2^-8 sum p |c - out| / sum p at the most, never outside of them, and exact where
// they are equal; its own rounding adds 2^-8 |out|. (Against 64 bits, 2-norms of all
// outputs: 64 requests of 8 nodes 2.1e-3, with the sum of weights in 32 bits 2.2e-3,
// their weights in 32 bits 1.7e-3, which is the outputs' own rounding.)
//
// Measured (512 + 64 columns, first launch + join): 64 requests of up to 8 nodes, 284
// in all, x 64 heads over up to 8192 keys, 182 + 16 us, 2326 clocks a tile of 64 rows: 1090 of
// the matrix cores and 1120 of LDS (265 KB at 236 bytes a clock), mostly in turn.
// 32 requests of one token x 64 heads over up to 65536 keys,
// 791 MB: 157 + 12 us, in the loop 6.1 TB/s, 3346 clocks a tile, the rows' way from
// HBM. One token over 4096 keys: 20 + 6.7 us, of which a walk's start (its request,
// pages, queries, first tile) takes 7, its end 4 and the place search 2.5. What did
// not carry: 64 keys a tile in a ring of two (282 us for the 64 requests), a running
// maximum with the sums rescaled (spills; 16 us more), rows permuted instead of
// padded (232 us), loads by global addresses (the compiler then waits for all of them).

template <int LC, bool WIN>
__global__ __launch_bounds__(512) void tree_bf16_kernel(Tree p, uint32_t min_per) {
    constexpr uint32_t NW = 8, ROWS = kRows16, PITCH = 256 * LC + kPad, NL = 4 * LC, NS = NL + 2, CT = 2 * LC, DR = 32 / NW;
    // the ring: separate objects, so that the compiler's own waits for DMA-written LDS stay per tile
    __shared__ __align__(1024) uint8_t ring0[kKT * (PITCH + 128)], ring1[kKT * (PITCH + 128)], ring2[kKT * (PITCH + 128)],
        ring3[kKT * (PITCH + 128)];
    constexpr uint32_t ROT = kKT * PITCH;  // the rotary parts' place behind the latent ones
    __shared__ __align__(1024) uint8_t pb0[ROWS * 64], pb1[ROWS * 64];  // weights [row][32 keys], of tiles in turn
    __shared__ float rowred[2][ROWS];                                   // per 16-key tile
    __shared__ uint64_t seen[ROWS];
    __shared__ uint32_t low[WIN ? ROWS : 1];  // the first key of each row's window
    __shared__ uint32_t flaws[kKT / 4];  // a byte per key of a tile with nodes: its row is not finite
    __shared__ uint32_t bad_page, again;
    __shared__ uint64_t tmp[2 * NW + 2 + kTries / 2];
    __shared__ Req found;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uni(tid >> 6), n = lane & 15u, g = lane >> 4;
    const uint32_t sr = 8u * (wave & ~1u), sk = 16u * (wave & 1u);  // first row and key of this wave's scores
    const uint32_t pr = 32u * (wave >> 2), wv = wave & 3u;          // first row of its sums, and its columns
    const uint32_t c = (blockIdx.x % 8u) * (kGrid / 8u) + blockIdx.x / 8u;
    const uint32_t H = p.a.n_heads, L = p.a.cache.kv_lora_rank, RP = p.a.cache.qk_rope;
    if (tid == 0) bad_page = again = 0;
    const Place f = find_place<ROWS, 64 * NW, kGrid, WIN>(p, c, min_per, tmp, (u32x2*)pb0, &found);
    if (tid < 2) p.desc[kDesc * (2 * c + tid)] = 0;
    Walks<ROWS, WIN> walks(p, f, c);
    if (!walks.more()) return;
    // the pages of a walk's first four tiles are read while the one before it ends
    int32_t ahead[4] = {0, 0, 0, 0};
    auto read_ahead = [&]() {
        if (walks.next.q.flaw) return;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) ahead[i] = walks.page(walks.next, walks.next.kt0 + i, DR * wave);
    };
    walks.find();
    read_ahead();
    for (;;) {
        const Walk w = walks.next;
        const Req& q = w.q;
        const uint32_t rt = w.rt, kt0 = w.kt0, kt1 = w.kt1, rows = walks.rows(w);

        f32x4 acc[2][CT];
        float m = kNone, l = 0.f;  // of row sr + n: the reference, this lane's part of the weights' sum
        auto clear = [&]() {
            l = 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (uint32_t k = 0; k < CT; k++) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        };
        bool bad = false;
        const bool more = walks.more();
        if (q.flaw) {
            clear();
        } else {
            auto page_of = [&](uint32_t t) { return walks.page(w, t, DR * wave); };
            // The wave's rows of tile t: one resource, whose bounds make zeros of rows
            // behind the last key. Tiles behind the walk's last are called for too, as
            // zeros, so that a wave's memory operations can be counted.
            const uint32_t stride = 2u * p.a.cache.row_stride;
            rsrc_t rs;
            auto find_rows = [&](uint32_t t, int32_t page_v) {
                const int32_t page = (int32_t)uni((uint32_t)page_v);
                const uint32_t key = key_of<WIN>(q, t) + DR * wave;
                const uint32_t left = t < kt1 && key < q.keys ? (q.keys - key < DR ? q.keys - key : DR) : 0u;
                const bool ok = page >= 0 && (uint32_t)page < p.a.cache.n_pages;
                bad |= left && !ok;
                const uint32_t row = ok ? ((uint32_t)page << p.psh) + (key & (p.a.cache.page_size - 1u)) : 0u;
                rs = make_rsrc((const uint8_t*)p.a.cache.d_rows + (uint64_t)row * stride,
                               ok && left ? (left - 1u) * stride + 2u * (L + RP) : 0u);
            };
            // lane's chunk of a latent part, and of the wave's rows' rotary parts
            const uint32_t lat_at = 8u * lane < L ? 16u * lane : kOOB;
            const uint32_t rot_i = lane >> 3, rot_ch = (lane & 7u) ^ swz8((DR * wave + rot_i) & 15u);
            const uint32_t rot_at = 8u * rot_ch < RP ? rot_i * stride + 2u * L + 16u * rot_ch : kOOB;
            auto issue_row = [&](uint8_t* lat, uint32_t i) {
                if (LC == 4 || lane < 16 * LC)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, WL_LDS(lat + (DR * wave + i) * PITCH), 16u, lat_at + i * stride,
                                                             0u, 0, 0);
            };
            auto issue_rot = [&](uint8_t* lat) {
                if (lane < 8 * DR)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, WL_LDS(lat + ROT + DR * wave * 128u), 16u, rot_at, 0u, 0, 0);
            };
            auto issue_tile = [&](uint8_t* lat, uint32_t t, int32_t page) {
                find_rows(t, page);
#pragma unroll
                for (uint32_t i = 0; i < DR; i++) issue_row(lat, i);
                issue_rot(lat);
            };
            int32_t page = 0, page1 = 0;  // of tiles t + 2 and t + 3
            // the queries of rows sr + n, in the operand's layout: lane (row n, k group g)
            bf16x8 qf[NS];
            auto read_queries = [&]() {
                const rsrc_t ql = make_rsrc((const uint16_t*)p.a.d_q_lat + q.t0 * p.a.q_lat_stride,
                                            2u * ((q.nodes - 1u) * (uint32_t)p.a.q_lat_stride + H * L));
                const rsrc_t qr = make_rsrc((const uint16_t*)p.a.d_q_rope + q.t0 * p.a.q_rope_stride,
                                            2u * ((q.nodes - 1u) * (uint32_t)p.a.q_rope_stride + H * RP));
                const uint32_t lr = sr + n, row = rt * ROWS + lr, node = row / H, h = row - node * H;
                const bool live = lr < rows;
                const uint32_t vl = live ? 2u * (node * (uint32_t)p.a.q_lat_stride + h * L + 8u * g) : kOOB;
                const uint32_t vr = live ? 2u * (node * (uint32_t)p.a.q_rope_stride + h * RP + 8u * g) : kOOB;
#pragma unroll
                for (uint32_t s = 0; s < NS; s++) {
                    u32x4 x = s < NL ? bld16(ql, vl + 64u * s, 0) : bld16(qr, vr + 64u * (s - NL), 0);
                    if (32u * (s < NL ? s : s - NL) + 8u * g >= (s < NL ? L : RP)) x = u32x4{0u, 0u, 0u, 0u};
                    qf[s] = as_bf16x8(x);
                }
                if (sk == 0 && g == 0) {
                    uint32_t from;
                    seen[lr] = sees<WIN>(p, q, live ? node : 0u, from);
                    if (WIN) low[lr] = from;
                }
            };
            auto has_nodes = [&](uint32_t t) {  // tree nodes, the end or a window's edge in tile t
                return is_masked<WIN>(p, q, key_of<WIN>(q, t), kKT);
            };
            // A row that some nodes may not see must not reach them through 0 x inf: in
            // a tile with nodes, those whose latent part is not finite are noted (their
            // scores will be NaN for those that see them) and the part is cleared. The
            // rotary part only enters scores. Each wave looks at the rows it called for.
            auto note_flaws = [&](uint8_t* lat, uint32_t t) {
                constexpr uint32_t LR = 64 / DR;  // lanes per row
                const uint32_t i = DR * wave + lane / LR;
                uint32_t nf = 0;
                if (WIN || t * kKT + i >= q.len) {
#pragma unroll 1
                    for (uint32_t k = lane % LR; k < 16 * LC; k += LR) {
                        u32x4* x = (u32x4*)(lat + i * PITCH + 16u * k);
                        if (has_nonfinite(*x)) {
                            nf = 1;
                            *x = u32x4{0u, 0u, 0u, 0u};
                        }
                    }
                }
                for (uint32_t d = 1; d < LR; d <<= 1) nf |= __shfl_xor(nf, d, 64);
                if (lane % LR == 0) ((uint8_t*)flaws)[i] = (uint8_t)nf;
            };
            // the key operand of step s: chunk 4 s + g of key row sk + n
            const uint32_t key_at = (sk + n) * PITCH + 16u * g, key_rot = (sk + n) * 128u + 16u * (g ^ swz8(n));
            auto kread = [&](const uint8_t* lat, uint32_t s) {
                return s < NL ? *(const u32x4*)(lat + key_at + 64u * s)
                              : *(const u32x4*)(lat + ROT + (key_rot ^ (64u * (s - NL))));
            };
            // the products of rows sr + n with keys sk + 4 g + j, in two sums
            auto products = [&](const uint8_t* lat, f32x4& s0, f32x4& s1) {
                constexpr uint32_t KP = 4;  // steps that the key operands are read ahead
                u32x4 kf[KP];
#pragma unroll
                for (uint32_t k = 0; k < KP; k++) kf[k] = kread(lat, k);
                s0 = s1 = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t s = 0; s < NS; s += 2) {
                    s0 = mma(as_bf16x8(kf[s % KP]), qf[s], s0);
                    s1 = mma(as_bf16x8(kf[(s + 1) % KP]), qf[s + 1], s1);
                    if (s + KP < NS) kf[s % KP] = kread(lat, s + KP);
                    if (s + 1 + KP < NS) kf[(s + 1) % KP] = kread(lat, s + 1 + KP);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // the scores in powers of two are s0 + s1 times the factor returned; those of
            // keys that the row does not see become -inf
            auto scores = [&](f32x4& s0, f32x4 s1, uint32_t t) {
#pragma unroll
                for (int k = 0; k < 4; k++) s0[k] += s1[k];
                if (!has_nodes(t)) return p.scale2;
                const uint32_t fl = flaws[sk / 4u + g];
                const uint64_t bits = seen[sr + n];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t key = key_of<WIN>(q, t) + sk + 4u * g + k;
                    const uint32_t bit = (uint32_t)(bits >> ((key - q.len) & 63u)) & (key < q.keys ? 1u : 0u);
                    const float nan = (fl >> (8 * k)) & 1u ? __builtin_nanf("") : 0.f;
                    const uint32_t old = key < q.len && (!WIN || key >= low[sr + n] || key < p.sinks) ? 1u : 0u;
                    s0[k] = ((WIN && key < q.len ? 0u : bit) | old) ? s0[k] * p.scale2 + nan : -INFINITY;
                }
                return 1.0f;
            };
            auto largest = [&](f32x4 x, float f) { return fmaxf(fmaxf(x[0] * f, x[1] * f), fmaxf(x[2] * f, x[3] * f)); };
            // m = the largest of x over the row's lanes and its two waves
            auto share_maxima = [&](float x) {
                x = fmaxf(x, __shfl_xor(x, 16, 64));
                x = fmaxf(x, __shfl_xor(x, 32, 64));
                if (g == 0) rowred[wave & 1u][sr + n] = x;
                ring_barrier();
                m = fmaxf(kNone, fmaxf(rowred[0][sr + n], rowred[1][sr + n]));
            };
            // through a window a row may see nothing of the first tile: the first of whose
            // keys it sees some sets its reference (its sums are zeros before)
            auto late_maxima = [&](float x) {
                const float before = m;
                share_maxima(x);
                if (before != kNone) m = before;
            };
            bool pass = false;
            uint32_t first = kt0;  // the tile that sets the reference
            // the value operand of columns 16 k of the wave's: lane group g has keys 4 g +
            // [0, 4) and 16 + 4 g + [0, 4)
            const uint32_t value_at = (4u * g + ((lane & 15u) >> 2)) * PITCH + 64u * LC * wv + 8u * (lane & 3u);
            auto vread = [&](const uint8_t* lat, uint32_t k) {
                const uint8_t* pa = lat + value_at + 32u * k;
                typedef __attribute__((address_space(3))) s16x4 l_s16x4;
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa + 16 * PITCH));
                const u32x2 xx = __builtin_bit_cast(u32x2, x), yy = __builtin_bit_cast(u32x2, y);
                return u32x4{xx[0], xx[1], yy[0], yy[1]};
            };
            // finds tile t's rows (its page came two tiles ago)
            auto next_rows = [&](uint32_t t) {
                find_rows(t, page);
                page = page1;
                page1 = page_of(t + 2);
            };
            // the weights, in the order of the values' keys: chunk g of a row
            const uint32_t put_at = (sr + n) * 64u + 16u * (g ^ swz4(n)) + sk / 2u;
            const uint32_t get_at = (pr + n) * 64u + 16u * (g ^ swz4(n));
            auto put_weights = [&](const float* e, uint8_t* pb) {
                const u32x2 x = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3])};
                *(u32x2*)(pb + put_at) = x;
                const float r[4] = {__uint_as_float(x[0] << 16), __uint_as_float(x[0] & 0xFFFF0000u),
                                    __uint_as_float(x[1] << 16), __uint_as_float(x[1] & 0xFFFF0000u)};
                l += (r[0] + r[1]) + (r[2] + r[3]);
                pass |= fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3])) > kMost;
            };
            // between two barriers: tile t - 1 is in b0 with weights w0, tile t in b1 with
            // weights w1 to be made, tile t + 2's place is b3; at t = kt1 the last sums
            auto turn = [&](uint8_t* b0, uint8_t* b1, uint8_t* b3, uint8_t* w0, uint8_t* w1, uint32_t t) {
                constexpr uint32_t VP = 2;  // column tiles that the values are read ahead
                u32x4 vf[VP];
                bf16x8 pf[2];
                const bool live = t < kt1;
                next_rows(t + 2);
                f32x4 s0, s1;
                float e[4], f;
                if (live) {
                    if (has_nodes(t)) {
                        note_flaws(b1, t);
                        ring_barrier();
                    }
                    products(b1, s0, s1);
                    if (WIN && has_nodes(t)) {
                        f = scores(s0, s1, t);
                        late_maxima(largest(s0, f));
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; i++) pf[i] = as_bf16x8(*(const u32x4*)(w0 + get_at + 1024u * i));
#pragma unroll
                for (uint32_t k = 0; k < VP; k++) vf[k] = vread(b0, k);
#pragma unroll
                for (uint32_t v = 0; v < CT; v++) {
#pragma unroll
                    for (int i = 0; i < 2; i++) acc[i][v] = mma(as_bf16x8(vf[v % VP]), pf[i], acc[i][v]);
                    if (v + VP < CT) vf[v % VP] = vread(b0, v + VP);
                    if (live) {
                        if (v == 0 && !(WIN && has_nodes(t))) f = scores(s0, s1, t);
                        if (v == 1) {
#pragma unroll
                            for (int k = 0; k < 4; k++) e[k] = exp2_(fmaf(s0[k], f, -m));
                        }
                        if (v == (CT == 2 ? 1 : 2)) put_weights(e, w1);
                    }
                    constexpr uint32_t PER = (DR + CT - 1) / CT;
#pragma unroll
                    for (uint32_t k = 0; k < DR; k++)
                        if (k >= v * PER && k < v * PER + PER) issue_row(b3, k);
                    if (v + 1 == CT) issue_rot(b3);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!live) return false;
                vm_wait<DR + 2>();  // tile t + 1 is there; t + 2 and a page may be on the way
                ring_barrier();
                return true;
            };
            for (;;) {
                clear();
                issue_tile(ring0, kt0, ahead[0]);
                issue_tile(ring1, kt0 + 1, ahead[1]);
                page = ahead[2];
                page1 = ahead[3];
                if (first == kt0) read_queries();
                vm_wait<0>();
                ring_barrier();
                if (has_nodes(kt0)) {
                    note_flaws(ring0, kt0);
                    ring_barrier();
                }
                next_rows(kt0 + 2);
#pragma unroll
                for (uint32_t i = 0; i < DR; i++) issue_row(ring2, i);
                issue_rot(ring2);
                {
                    f32x4 s0, s1;
                    products(ring0, s0, s1);
                    const float f = scores(s0, s1, kt0);
                    if (first == kt0) share_maxima(largest(s0, f));
                    float e[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) e[k] = exp2_(fmaf(s0[k], f, -m));
                    put_weights(e, pb0);
                }
                vm_wait<DR + 2>();
                ring_barrier();
                for (uint32_t t = kt0 + 1;; t += 4) {
                    if (!turn(ring0, ring1, ring3, pb0, pb1, t)) break;
                    if (!turn(ring1, ring2, ring0, pb1, pb0, t + 1)) break;
                    if (!turn(ring2, ring3, ring1, pb0, pb1, t + 2)) break;
                    if (!turn(ring3, ring0, ring2, pb1, pb0, t + 3)) break;
                }
                vm_wait<0>();
                if (first != kt0) break;
#pragma unroll
                for (uint32_t i = 0; i < 2; i++) pass |= pr + 16u * i + n < rows && nonfinite(acc[i]);
                if (__ballot(pass) && lane == 0) again = 1u;
                ring_barrier();
                const bool redo = uni(again) != 0;
                ring_barrier();
                if (!redo) break;
                if (tid == 0) again = 0u;
                float x = kNone;
                for (uint32_t t = kt0; t < kt1; t++) {
                    issue_tile(ring0, t, page_of(t));
                    vm_wait<0>();
                    ring_barrier();
                    note_flaws(ring0, t);
                    ring_barrier();
                    f32x4 s0, s1;
                    products(ring0, s0, s1);
                    const float f = scores(s0, s1, t);
                    x = fmaxf(x, largest(s0, f));
                    ring_barrier();
                }
                share_maxima(x);
                m += lift_of((kt1 - kt0) * kKT);
                ring_barrier();
                first = ~0u;
            }
        }
        if (more) {
            walks.find();
            read_ahead();
        }
        // the weights' sums over the row's lanes and waves; flaws
        if (__ballot(bad) && lane == 0) {
            bad_page = 1u;
            set_status(p.a.d_status, WL_PAGED_E_PAGE);
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0) rowred[wave & 1u][sr + n] = l;
        const bool whole = kt1 - kt0 == q.nkt;
        if (!whole && sk == 0 && g == 0) p.part_ml[2u * (w.slot * ROWS + sr + n)] = m;
        ring_barrier();
        const bool nan = bad_page != 0 || q.flaw;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t lr = pr + 16u * i + n;
            float sum = rowred[0][lr] + rowred[1][lr];
            if (nan) sum = __builtin_nanf("");
            if (lr < rows) {
                put_row<ROWS, LC, true, CT>(p, w, whole, lr, sum, acc[i], 32u * LC * wv + 4u * g);
                if (!whole && wv == 0 && g == 0) p.part_ml[2u * (w.slot * ROWS + lr) + 1u] = sum;
            }
        }
        if (!whole && tid == (w.slot & 1u)) walks.name_part(w);  // the thread that cleared it
        if (!more) return;
        ring_barrier();
        if (tid == 0) bad_page = 0u;
        ring_barrier();
    }
}

// ---- 32-bit queries -------------------------------------------------------------
// A 32-bit value is the sum of three bf16 ones, h + m + l, each the rounding of what
// the ones before it leave (which is exact: 24 bits, then 16, then 8), m at most 2^-8
// of the value and l 2^-16. A product of two such sums is, but for its m l, l m and
// l l, together 2^-23 of it at the most and of either sign, the six products
// h h, h m, m h, m m, h l, l h; of a bf16 value and such a sum, all of three: exact
// products in the matrix cores, summed in f32, the scores' leading ones apart from
// the others.
//
// 32 rows against 32 keys (WIDE, a cache of 32-bit rows: 16) at a time, four waves.
// The next tile's rows are read into registers while this one is worked on, then cut
// up into LDS. Scores: a wave has 16 rows' queries, half of their columns, and adds
// its sums to those of the wave with the other half, so a row's three parts take 108
// registers; with the sums (64) and the next rows (36) that is what two work-groups a
// CU leave a wave. They are what overlaps: one's products run while the other cuts,
// takes exponentials or waits. (All columns in one wave and one work-group a CU,
// first: one request of 64 nodes x 64 heads over 8192 keys 278 us, 5 requests of 7
// nodes over up to 2000 32-bit rows 75 us; so, 242 and 58 us.) Values: 16 columns of
// all rows at once. Of 16 keys, the 32 places of a product hold two parts of each:
// (h, m) against the weights' (h, h) and (m, m), (h, l) against (l, h).
// Lane addresses are computed where they are used (afresh): held, they spill. (With 512
// columns 2 registers a lane still do, 8 in WIDE.)
//
// Bound by the matrix cores: 102 (WIDE 102 of 16 keys) products a wave and tile, 16
// clocks each. The 64 nodes' 73 GFLOP, three products each, take 181 us at the rate
// of a large library product (1211 TFLOP/s), 207 to 217 us with the joining here
// (cards differ), 11 of them for the queries' reads at the start and 12 for the join.
// Reading the next rows a piece at a time between the scores' products made no
// difference. Rows of 4 bits are read as they lie in the cache and brought to bf16, which
// holds them, on their way into LDS: 5 requests of up to 7 nodes (16 in all) over up to 2000
// keys 34 us, of which the join takes 9 and a walk's start and end most.
WL_DEV void cut3(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {  // two values' parts, x in the low halves
    auto low = [](uint32_t v) { return __uint_as_float(v << 16); };
    auto high = [](uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); };
    h = pack_bf16(x, y);
    x -= low(h), y -= high(h);
    m = pack_bf16(x, y);
    l = pack_bf16(x - low(m), y - high(m));
}
WL_DEV bool nonfinite(float x) { return (__float_as_uint(x) & 0x7F800000u) == 0x7F800000u; }

// The cache that 32-bit queries meet: 32-bit rows (WIDE), 16-bit ones, or 4-bit ones.
enum : int { kCacheF32 = 0, kCacheBf16 = 1, kCacheMx4 = 2 };
template <int LC, int CK, bool WIN>
__global__ __launch_bounds__(256, 2) void tree_f32_kernel(Tree p, uint32_t min_per) {
    constexpr bool WIDE = CK == kCacheF32, MX = CK == kCacheMx4;
    constexpr uint32_t ROWS = kRows32, KT = WIDE ? 16 : 32, PITCH = 256 * LC + kPad, NL = 4 * LC, NH = NL / 2 + 1, CT = 2 * LC;
    constexpr uint32_t DR = KT / 4, NK = KT / 8, NP = WIDE ? 3 : 1, ROT = KT * PITCH, PIECE = ROT + KT * 128, ES = WIDE ? 4 : 2;
    __shared__ __align__(1024) uint8_t tile[NP * PIECE];
    __shared__ __align__(1024) uint8_t pb[3 * ROWS * 64];  // weights [operand][row][32 places]
    __shared__ __align__(16) float other[4][64][NK];     // scores over half of the columns, for the wave of the others
    __shared__ float rowred[2][ROWS];
    __shared__ uint64_t seen[ROWS];
    __shared__ uint32_t low[WIN ? ROWS : 1];
    __shared__ uint32_t flaws[KT / 4];
    __shared__ uint32_t bad_page, again;
    __shared__ uint64_t tmp[2 * 4 + 2 + kTries / 2];
    __shared__ Req found;
    const uint32_t tid = threadIdx.x, wave = uni(tid >> 6);
    // the wave's scores: rows sr + n, over the 32-column slices NH hf .. of all of the
    // tile's keys; it ends up with half of those keys
    const uint32_t sr = 8u * (wave & ~1u), hf = wave & 1u;
    const uint32_t c = (blockIdx.x % 8u) * (kGridF32 / 8u) + blockIdx.x / 8u;
    const uint32_t H = p.a.n_heads, L = p.a.cache.kv_lora_rank, RP = p.a.cache.qk_rope;
    if (tid == 0) bad_page = again = 0;
    const Place f = find_place<ROWS, 256, kGridF32, WIN>(p, c, min_per, tmp, (u32x2*)pb, &found);
    if (tid < 2) p.desc[kDesc * (2 * c + tid)] = 0;
    Walks<ROWS, WIN> walks(p, f, c);
    if (!walks.more()) return;
    for (;;) {
        walks.find();
        const Walk w = walks.next;
        const Req& q = w.q;
        const uint32_t kt0 = w.kt0, kt1 = w.kt1, rows = walks.rows(w);
        f32x4 acc[2][CT];
        float m = kNone, l = 0.f;
        auto clear = [&]() __attribute__((always_inline)) {
            l = 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (uint32_t k = 0; k < CT; k++) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        };
        bool bad = false;
        if (q.flaw) {
            clear();
        } else {
            // the wave's DR rows of a tile, in registers: chunk i 64 + lane of their latent
            // parts (EL to a row), then of their rotary ones (ER)
            // (4-bit rows: 32 values a chunk, with their scale byte, and 16-bit rotary parts)
            constexpr uint32_t EL = MX ? 4 * LC : 8 * ES * LC, NLAT = (DR * EL + 63) / 64, ER = 4 * ES, NROT = DR * ER / 64;
            const uint32_t stride = (MX ? 1u : ES) * p.a.cache.row_stride;
            const uint32_t rot0 = MX ? L / 2u + kMxScales : ES * L;  // where a row's rotary part begins
            u32x4 raw[NLAT + NROT];
            uint32_t mx[MX ? NLAT : 1];
            // the first key of tile t (of KT keys)
            auto first_key = [&](uint32_t t) { return key_of<WIN>(q, t / (kKT / KT)) + t % (kKT / KT) * KT; };
            auto page_of = [&](uint32_t t) __attribute__((always_inline)) {  // of its rows in tile t (pages have at least 8)
                const uint32_t key = first_key(t) + DR * wave;
                return p.a.d_table[(size_t)w.r * p.a.max_pages + ((key < q.keys ? key : q.keys - 1u) >> p.psh)];
            };
            int32_t next_page;  // of the next tile to read
            auto read_tile = [&](uint32_t t) __attribute__((always_inline)) {
                const uint32_t lane = afresh(tid) & 63u;
                const int32_t page = (int32_t)uni((uint32_t)next_page);
                const uint32_t key = first_key(t) + DR * wave;
                const uint32_t left = key < q.keys ? (q.keys - key < DR ? q.keys - key : DR) : 0u;
                const bool ok = page >= 0 && (uint32_t)page < p.a.cache.n_pages;
                bad |= left && !ok;
                const uint32_t row = ok ? ((uint32_t)page << p.psh) + (key & (p.a.cache.page_size - 1u)) : 0u;
                const rsrc_t rs = make_rsrc((const uint8_t*)p.a.cache.d_rows + (uint64_t)row * stride,
                                            ok && left ? (left - 1u) * stride + rot0 + ES * RP : 0u);
                next_page = page_of(t + 1);
#pragma unroll
                for (uint32_t i = 0; i < NLAT; i++) {
                    const uint32_t e = 64u * i + lane, k = e % EL;
                    // row j of whole chunks in the scalar offset (the first one's again for those
                    // behind the last key, which no row of scores sees), not in address registers
                    const uint32_t j = i / (EL < 64 ? 1 : EL / 64);
                    if (MX) {
                        const bool has = 32u * k < L && e / EL < DR;
                        raw[i] = bld16(rs, has ? (e / EL) * stride + 16u * k : kOOB, 0);
                        mx[i] = bld1(rs, has ? (e / EL) * stride + L / 2u + mx_scale_at(k) : kOOB, 0);
                    } else if (EL < 64) raw[i] = bld16(rs, 16u * k < ES * L ? (e / EL) * stride + 16u * k : kOOB, 0);
                    else raw[i] = bld16(rs, 16u * k < ES * L ? 16u * k : kOOB, j < left ? j * stride : 0u);
                }
#pragma unroll
                for (uint32_t i = 0; i < NROT; i++) {
                    const uint32_t e = 64u * i + lane, k = e % ER;
                    raw[NLAT + i] = bld16(rs, 16u * k < ES * RP ? (e / ER) * stride + rot0 + 16u * k : kOOB, 0);
                }
            };
            auto has_nodes = [&](uint32_t t) { return is_masked<WIN>(p, q, first_key(t), KT); };  // as above
            // into LDS, in parts; of rows of nodes what is not finite is noted and cleared
            // (their scores will be NaN for those that see them)
            auto stage = [&](uint32_t t) __attribute__((always_inline)) {
                const uint32_t lane = afresh(tid) & 63u;
                auto put = [&](u32x4 x, uint32_t at) {
                    if (WIDE) {
                        uint32_t v[3][2];
#pragma unroll
                        for (int k = 0; k < 2; k++)
                            cut3(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1]), v[0][k], v[1][k], v[2][k]);
#pragma unroll
                        for (uint32_t j = 0; j < NP; j++) *(u32x2*)(tile + j * PIECE + at) = u32x2{v[j][0], v[j][1]};
                    } else {
                        *(u32x4*)(tile + at) = x;
                    }
                };
                if (has_nodes(t)) {
#pragma unroll
                    for (uint32_t i = 0; i < NLAT + NROT; i++) {
                        const uint32_t e = 64u * (i < NLAT ? i : i - NLAT) + lane, row = DR * wave + e / (i < NLAT ? EL : ER);
                        bool nf = false;
                        if (MX && i < NLAT) {
                            nf = mx[i] > kMxHi;
                        } else if (WIDE) {
#pragma unroll
                            for (int j = 0; j < 4; j++) nf |= nonfinite(__uint_as_float(raw[i][j]));
                        } else {
                            nf = has_nonfinite(raw[i]);
                        }
                        if (nf && (WIN || t * KT + row >= q.len)) {
                            ((uint8_t*)flaws)[row] = 1;
                            raw[i] = u32x4{0u, 0u, 0u, 0u};
                            if (MX && i < NLAT) mx[i] = 0;
                        }
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < NLAT + NROT; i++) {
                    const bool lat = i < NLAT;
                    const uint32_t e = 64u * (lat ? i : i - NLAT) + lane, k = e % (lat ? EL : ER);
                    const uint32_t row = DR * wave + e / (lat ? EL : ER);
                    if (MX && lat) {
                        if (e / EL < DR) {
                            const MxBlock b = mx_block(raw[i], mx[i], k >> 2);
#pragma unroll
                            for (uint32_t j = 0; j < 4; j++) mx_put(b, j, tile + row * PITCH + 64u * k);
                            if (mx[i] > kMxHi) *(u32x4*)(tile + row * PITCH + 64u * k) = u32x4{~0u, ~0u, ~0u, ~0u};  // NaN, and so its scores
                        }
                        continue;
                    }
                    const uint32_t b = WIDE ? 8u * k : 16u * k;  // of a bf16 row
                    put(raw[i], lat ? row * PITCH + b : ROT + row * 128u + (b ^ (16u * swz8(row & 15u))));
                }
            };
            // the queries of rows sr + n, in parts, in the operand's layout: lane (row n, k group g);
            // slice s of the row's 2 NH: of the latent part's 32 columns each, and the rotary one's last two
            bf16x8 qf[3][NH];
            struct Queries {
                u32x4 x[NH][2];
            };
            auto read_queries = [&](Queries& f) __attribute__((always_inline)) {
                const rsrc_t ql = make_rsrc((const float*)p.a.d_q_lat + q.t0 * p.a.q_lat_stride,
                                            4u * ((q.nodes - 1u) * (uint32_t)p.a.q_lat_stride + H * L));
                const rsrc_t qr = make_rsrc((const float*)p.a.d_q_rope + q.t0 * p.a.q_rope_stride,
                                            4u * ((q.nodes - 1u) * (uint32_t)p.a.q_rope_stride + H * RP));
                const uint32_t ln = afresh(tid) & 63u, g = ln >> 4;
                const uint32_t lr = sr + (ln & 15u), row = w.rt * ROWS + lr, node = row / H, h = row - node * H;
                const bool live = lr < rows;
                const uint32_t vl = 4u * (node * (uint32_t)p.a.q_lat_stride + h * L);
                const uint32_t vr = 4u * (node * (uint32_t)p.a.q_rope_stride + h * RP);
#pragma unroll
                for (uint32_t i = 0; i < NH; i++) {
                    const bool rot = i + 1 == NH;  // the last of each half is a rotary one
                    const uint32_t col = 32u * (rot ? hf : (NH - 1u) * hf + i) + 8u * g;
                    const uint32_t at = live && col < (rot ? RP : L) ? (rot ? vr : vl) + 4u * col : kOOB;
#pragma unroll
                    for (uint32_t k = 0; k < 2; k++) f.x[i][k] = bld16(rot ? qr : ql, at, 16u * k);
                }
            };
            auto cut_queries = [&](const Queries& f) __attribute__((always_inline)) {
#pragma unroll
                for (uint32_t i = 0; i < NH; i++) {
                    u32x4 part[3];
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) {
                        uint32_t v[3];
                        const u32x4 x = f.x[i][k >> 1];
                        cut3(__uint_as_float(x[2 * (k & 1)]), __uint_as_float(x[2 * (k & 1) + 1]), v[0], v[1], v[2]);
#pragma unroll
                        for (int j = 0; j < 3; j++) part[j][k] = v[j];
                    }
#pragma unroll
                    for (int j = 0; j < 3; j++) qf[j][i] = as_bf16x8(part[j]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                const uint32_t ln = afresh(tid) & 63u, lr = sr + (ln & 15u);
                if (hf == 0 && (ln >> 4) == 0) {
                    uint32_t from;
                    seen[lr] = sees<WIN>(p, q, lr < rows ? (w.rt * ROWS + lr) / H : 0u, from);
                    if (WIN) low[lr] = from;
                }
            };
            // the scores in powers of two of row sr + n with keys own_keys(g) + k, -inf where unseen
            constexpr uint32_t NB = KT / 16;
            auto own_keys = [&](uint32_t g) { return WIDE ? 4u * g + 2u * hf : 16u * hf + 4u * g; };
            struct Sc {
                float v[NK];
            };
            auto scores = [&](uint32_t t) __attribute__((always_inline)) {
                const uint32_t lane = afresh(tid) & 63u, n = lane & 15u, g = lane >> 4;
                const uint32_t key_at = n * PITCH + 64u * (NH - 1u) * hf + 16u * g;
                const uint32_t key_rot = ROT + n * 128u + ((16u * (g ^ swz8(n))) ^ (64u * hf));
                auto kread = [&](uint32_t i, uint32_t piece, uint32_t block) __attribute__((always_inline)) {
                    return as_bf16x8(i + 1 < NH ? *(const u32x4*)(tile + PIECE * piece + 16u * block * PITCH + key_at + 64u * i)
                                                : *(const u32x4*)(tile + PIECE * piece + 2048u * block + key_rot));
                };
                const uint32_t own = own_keys(g);
                f32x4 s0[NB], s1[NB];
#pragma unroll
                for (uint32_t b = 0; b < NB; b++) s0[b] = s1[b] = f32x4{0.f, 0.f, 0.f, 0.f};
                bf16x8 kf[2][NB][NP];
                auto kread_all = [&](uint32_t i) __attribute__((always_inline)) {
#pragma unroll
                    for (uint32_t b = 0; b < NB; b++)
#pragma unroll
                        for (uint32_t j = 0; j < NP; j++) kf[i & 1u][b][j] = kread(i, j, b);
                };
                kread_all(0);
#pragma unroll
                for (uint32_t i = 0; i < NH; i++) {
                    if (i + 1 < NH) kread_all(i + 1);
#pragma unroll
                    for (uint32_t k = 0; k < (WIDE ? 6 : 3); k++) {
#pragma unroll
                        for (uint32_t b = 0; b < NB; b++) {
                            const bf16x8* kp = kf[i & 1u][b];
                            // h h apart; then h l, (l h, m m, m h,) h m
                            if (k == 0) s0[b] = mma(kp[0], qf[0][i], s0[b]);
                            else if (k == 1) s1[b] = mma(kp[0], qf[2][i], s1[b]);
                            else if (k == (WIDE ? 5 : 2)) s1[b] = mma(kp[0], qf[1][i], s1[b]);
                            else if (k == 2) s1[b] = mma(kp[NP - 1], qf[0][i], s1[b]);
                            else s1[b] = mma(kp[NP > 1 ? 1 : 0], qf[k == 3 ? 1 : 0][i], s1[b]);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                Sc sc;
                if (WIDE) {
                    const f32x4 y = s0[0] + s1[0];
#pragma unroll
                    for (uint32_t k = 0; k < NK; k++) {
                        sc.v[k] = hf ? y[2 + k] : y[k];
                        other[wave][lane][k] = hf ? y[k] : y[2 + k];
                    }
                } else {
                    const f32x4 a = s0[0] + s1[0], b = s0[NB - 1] + s1[NB - 1];
#pragma unroll
                    for (uint32_t k = 0; k < NK; k++) {
                        sc.v[k] = hf ? b[k] : a[k];
                        other[wave][lane][k] = hf ? a[k] : b[k];
                    }
                }
                ring_barrier();
#pragma unroll
                for (uint32_t k = 0; k < NK; k++) sc.v[k] = (sc.v[k] + other[wave ^ 1u][lane][k]) * p.scale2;
                if (has_nodes(t)) {
                    const uint64_t bits = seen[sr + n];
#pragma unroll
                    for (uint32_t k = 0; k < NK; k++) {
                        const uint32_t key = first_key(t) + own + k;
                        const uint32_t bit = (uint32_t)(bits >> ((key - q.len) & 63u)) & (key < q.keys ? 1u : 0u);
                        const float nan = ((const uint8_t*)flaws)[own + k] ? __builtin_nanf("") : 0.f;
                        const uint32_t old = key < q.len && (!WIN || key >= low[sr + n] || key < p.sinks) ? 1u : 0u;
                        sc.v[k] = ((WIN && key < q.len ? 0u : bit) | old) ? sc.v[k] + nan : -INFINITY;
                    }
                }
                return sc;
            };
            auto largest = [&](const Sc& x) {
                return WIDE ? fmaxf(x.v[0], x.v[1]) : fmaxf(fmaxf(x.v[0], x.v[1]), fmaxf(x.v[NK - 2], x.v[NK - 1]));
            };
            auto share_maxima = [&](float x) {
                const uint32_t lane = afresh(tid) & 63u, n = lane & 15u, g = lane >> 4;
                x = fmaxf(x, __shfl_xor(x, 16, 64));
                x = fmaxf(x, __shfl_xor(x, 32, 64));
                if (g == 0) rowred[wave & 1u][sr + n] = x;
                ring_barrier();
                m = fmaxf(kNone, fmaxf(rowred[0][sr + n], rowred[1][sr + n]));
            };
            // 16 columns' values against 32 places of the weights: of KT = 32 keys, or of 16
            // keys in their first part and in part j
            auto vread = [&](uint32_t value_at, uint32_t k, uint32_t j) __attribute__((always_inline)) {
                const uint8_t* pa = tile + value_at + 32u * k;
                typedef __attribute__((address_space(3))) s16x4 l_s16x4;
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa + (WIDE ? j * PIECE : 16 * PITCH)));
                const u32x2 xx = __builtin_bit_cast(u32x2, x), yy = __builtin_bit_cast(u32x2, y);
                return as_bf16x8(u32x4{xx[0], xx[1], yy[0], yy[1]});
            };
            // the weights e of row sr + n in places: parts h, m, l against 32 keys; or
            // against a key's value parts (h, m): h h and m m; against its (h, l): l h
            auto put_weights = [&](uint32_t put_at, const uint32_t (&e)[3][NK / 2]) __attribute__((always_inline)) {
#pragma unroll
                for (uint32_t j = 0; j < 3; j++) {
                    uint8_t* o = pb + j * ROWS * 64u + put_at;
                    if (WIDE) {
                        *(uint32_t*)(o + 4u * hf) = e[j][0];
                        *(uint32_t*)(o + 4u * hf + 8u) = j < 2 ? e[j][0] : e[0][0];
                    } else {
                        *(u32x2*)(o + 8u * hf) = u32x2{e[j][0], e[j][NK / 2 - 1]};
                    }
                }
            };
            bool pass = false;
            // a walk; SUMS false: over the scores alone, for their maxima
            auto go = [&](bool known, auto sums) __attribute__((always_inline)) {
                constexpr bool SUMS = decltype(sums)::value;
                float x = kNone;
                const uint32_t t0 = kt0 * (kKT / KT), t1 = kt1 * (kKT / KT);
                next_page = page_of(t0);
                Queries first;
                if (SUMS && !known) read_queries(first);
                __builtin_amdgcn_sched_barrier(0);
                read_tile(t0);
                if (SUMS && !known) cut_queries(first);
                if (SUMS) clear();
                for (uint32_t t = t0; t < t1; t++) {
                    if (has_nodes(t)) {
                        if (const uint32_t i = afresh(tid); i < KT / 4) flaws[i] = 0;
                        ring_barrier();
                    }
                    stage(t);
                    ring_barrier();
                    const Sc sc = scores(t);
                    if (t + 1 < t1) read_tile(t + 1);
                    if (SUMS) {
                        if (t == t0 && !known) share_maxima(largest(sc));
                        else if (WIN && has_nodes(t)) {  // the first tile of whose keys a row sees some, as above
                            const float before = m;
                            share_maxima(largest(sc));
                            if (before != kNone) m = before;
                        }
                        float top = 0.f;
                        uint32_t e[3][NK / 2];
#pragma unroll
                        for (uint32_t k = 0; k < NK / 2; k++) {
                            const float v = exp2_(sc.v[2 * k] - m), v1 = exp2_(sc.v[2 * k + 1] - m);
                            l += v + v1;
                            top = fmaxf(top, fmaxf(v, v1));
                            cut3(v, v1, e[0][k], e[1][k], e[2][k]);
                        }
                        pass |= top > kMost;
                        const uint32_t lane = afresh(tid) & 63u, n = lane & 15u, g = lane >> 4;
                        const uint32_t put_at = (sr + n) * 64u + 16u * (g ^ swz4(n)), get_at = n * 64u + 16u * (g ^ swz4(n));
                        const uint32_t value_at = (4u * g + (n >> 2)) * PITCH + 64u * LC * wave + 8u * (n & 3u);
                        put_weights(put_at, e);
                        ring_barrier();
                        bf16x8 pf[3][2];
#pragma unroll
                        for (uint32_t j = 0; j < 3; j++)
#pragma unroll
                            for (int i = 0; i < 2; i++)
                                pf[j][i] = as_bf16x8(*(const u32x4*)(pb + j * ROWS * 64u + get_at + 1024u * i));
                        bf16x8 va[2], vb[2];
                        auto vread_all = [&](uint32_t v) __attribute__((always_inline)) {
                            va[v & 1u] = vread(value_at, v, 1);
                            vb[v & 1u] = WIDE ? vread(value_at, v, 2) : va[v & 1u];
                        };
                        vread_all(0);
#pragma unroll
                        for (uint32_t v = 0; v < CT; v++) {
                            if (v + 1 < CT) vread_all(v + 1);
                            f32x4 y[2];
#pragma unroll
                            for (int i = 0; i < 2; i++) y[i] = mma(vb[v & 1u], pf[2][i], acc[i][v]);
#pragma unroll
                            for (int i = 0; i < 2; i++) y[i] = mma(va[v & 1u], pf[1][i], y[i]);
#pragma unroll
                            for (int i = 0; i < 2; i++) acc[i][v] = mma(va[v & 1u], pf[0][i], y[i]);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    } else {
                        x = fmaxf(x, largest(sc));
                    }
                    ring_barrier();
                }
                return x;
            };
            using Sums = std::integral_constant<bool, true>;
            using Maxima = std::integral_constant<bool, false>;
            go(false, Sums{});
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) pass |= 16u * i + (afresh(tid) & 15u) < rows && nonfinite(acc[i]);
            if (__ballot(pass) && (tid & 63u) == 0) again = 1u;
            ring_barrier();
            const bool redo = uni(again) != 0;
            ring_barrier();
            if (redo) {
                if (tid == 0) again = 0u;
                share_maxima(go(true, Maxima{}));
                m += lift_of((kt1 - kt0) * kKT);
                go(true, Sums{});
            }
        }
        if (__ballot(bad) && (tid & 63u) == 0) {
            bad_page = 1u;
            set_status(p.a.d_status, WL_PAGED_E_PAGE);
        }
        const uint32_t lane = afresh(tid) & 63u, n = lane & 15u, g = lane >> 4;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0) rowred[wave & 1u][sr + n] = l;
        const bool whole = kt1 - kt0 == q.nkt;
        if (!whole && hf == 0 && g == 0) p.part_ml[2u * (w.slot * ROWS + sr + n)] = m;
        ring_barrier();
        const bool nan = bad_page != 0 || q.flaw;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t lr = 16u * i + n;
            float sum = rowred[0][lr] + rowred[1][lr];
            if (nan) sum = __builtin_nanf("");
            if (lr < rows) {
                put_row<ROWS, LC, false, CT>(p, w, whole, lr, sum, acc[i], 32u * LC * wave + 4u * g);
                if (!whole && wave == 0 && g == 0) p.part_ml[2u * (w.slot * ROWS + lr) + 1u] = sum;
            }
        }
        if (!whole && tid == (w.slot & 1u)) walks.name_part(w);  // the thread that cleared it
        if (!walks.more()) return;
        ring_barrier();
        if (tid == 0) bad_page = 0u;
        ring_barrier();
    }
}
template <int LC, bool WIN>
int run_bf16(const Tree& p, hipStream_t st) {
    hipLaunchKernelGGL((tree_bf16_kernel<LC, WIN>), dim3(kGrid), dim3(512), 0, st, p, kMinPer);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL((tree_join_kernel<kGrid, kRows16, LC, true>), dim3(2 * kGrid, 4), dim3(256), 0, st, p);
    return (int)hipGetLastError();
}

template <int LC, int CK, bool WIN>
int run_f32(const Tree& p, hipStream_t st) {
    hipLaunchKernelGGL((tree_f32_kernel<LC, CK, WIN>), dim3(kGridF32), dim3(256), 0, st, p, kMinPer);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL((tree_join_kernel<kGridF32, kRows32, LC, false>), dim3(2 * kGridF32, 2), dim3(256), 0, st, p);
    return (int)hipGetLastError();
}

template <bool WIN>
int launch(const Tree& p, hipStream_t st) {
    return by_class(p.a, [&](auto lc) {
        constexpr int LC = decltype(lc)::value;
        if (p.a.dtype == WL_TYPE_BF16) return run_bf16<LC, WIN>(p, st);
        return p.a.cache.dtype == WL_TYPE_MXFP4  ? run_f32<LC, kCacheMx4, WIN>(p, st)
               : p.a.cache.dtype == WL_TYPE_BF16 ? run_f32<LC, kCacheBf16, WIN>(p, st)
                                                 : run_f32<LC, kCacheF32, WIN>(p, st);
    });
}
}  // namespace

size_t tree_scratch(const wl_tree_attn& a) {
    return part_rows(a) * (128 * lat_class(a) + 2) * 4 + 2 * kGridF32 * kDesc * 4;
}

int launch_tree(const wl_tree_attn& a, uint32_t window, uint32_t sinks, void* stream) {
    if (a.dtype == WL_TYPE_BF16 && a.cache.dtype == WL_TYPE_MXFP4) return launch_tree_mx4(a, window, sinks, stream);
    const Tree p = make_tree(a, window, sinks);
    return window ? launch<true>(p, (hipStream_t)stream) : launch<false>(p, (hipStream_t)stream);
}

}  // namespace paged
}  // namespace wl
