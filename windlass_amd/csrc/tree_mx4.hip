// tree_mx4.hip — attention of trees of drafted tokens, 16-bit queries over a paged
// cache of 4-bit rows (wl_paged_tree_attention, wl_paged_window_attention).
#include <hip/hip_runtime.h>

#include "tree_dev.h"

namespace wl {
namespace paged {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(6))) uint32_t u32x6;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(32))) float f32x32;

// ---- 16-bit queries, 4-bit rows --------------------------------------------------
// As over 16-bit rows (tree_attn.hip: a reference instead of a running maximum, weights
// in bf16 divided by the sum of what they are then, a walk done again where weights pass
// kMost), with 64 rows (node, head) against 32 keys at a time by eight waves:
//   S^T[keys][rows] = K Q^T: wave w takes rows 16 (w / 2) and keys 16 (w % 2). The values
//           meet the scaled products as they lie in the cache, 128 columns at a time with
//           their blocks' scales; the queries, in bf16, are cut into three pieces of 6 bits
//           each (E2M3) with scales of their own per 32 columns: a piece has 4 leading bits
//           and takes 4 to 5 bits of what is left, so 14 below the block's largest value, all
//           8 bits of a query that is at least a 120th of it. Their products and sums are
//           f32. The rotary part is a product in bf16.
//   O^T[cols][rows] += V^T P^T: the tile's values are brought to bf16 (which holds them
//           exactly) once for all waves, in LDS, and read transposed: wave w has columns
//           [16 LC w, + 16 LC) of all rows. (Scaled products here would need the weights in
//           pieces too, and the values transposed in halves of bytes.)
// A row is 400 bytes instead of 1152, so what bounds this is not memory but the CU: a
// tile is some 2200 clocks, of which products take 760 to 1000 and LDS some 1050 (a tile
// comes in, is read as keys, by its wave's lanes once more for conversion, written in
// bf16, read transposed), the rest is waits at the turn's one barrier; a work-group a
// CU has two waves a SIMD to fill them. Hence: a ring of four tiles, three on the way;
// operands read ahead of their products, values converted between the scores' products,
// LDS rows and chunks placed so that no access meets a bank twice, a walk's addresses
// found 64 tiles at a time.
// Measured (512 + 64 columns, both launches): 32 requests of one token x 64 heads over
// up to 65536 keys (22775 on average, 296 MB) 121 to 130 us (cards differ), 780 to 840
// TFLOP/s or 54 to 58 % of a large bf16 product's rate (over 16-bit rows 170); 64 of up to 8
// nodes (279 in all) over up to 8192 164 to 171 us, 590 to 610 TFLOP/s (198 to 201); one token over
// 4096 keys 26, all of it latencies (28).
// Two pieces of the queries instead of three would be 6 % faster and lose 5 of the 14
// bits. Without effect: the two waves of a SIMD in opposite order, wave priorities, values
// read before the barrier.

// Pieces of 32 queries that meet one scale of a key: q = sum of p_i 2^s_i, p_i of E2M3;
// s_1 puts the largest into (3.75, 7.5], the others fall by 4 and 9 powers of two.
constexpr uint32_t kQueryPieces = 3;  // (they are moved as three)

template <int LC, bool WIN>
__global__ __launch_bounds__(512) void tree_mx4_kernel(Tree p, uint32_t min_per) {
    constexpr uint32_t NW = 8, ROWS = kRows16, PITCH = 256 * LC + kPad, CT = LC, DR = 32 / NW, QP = kQueryPieces, NB = 4 * LC;
    // a tile as it comes: 256 bytes of values a row, chunk c at c ^ swap(row); then by
    // wave its rows' rotary parts, chunk c at c ^ swz8(row), and scales, behind 64 bytes a
    // wave (1 KB, so that all lanes take part: loads under a condition the compiler cannot
    // count, and waits for)
    constexpr uint32_t AUX = kKT * 256, AUXW = 1024, RAW = AUX + NW * AUXW;
    static_assert(ROWS * NB * 64 <= 2 * kKT * PITCH && ROWS * NB * 8 <= RAW, "the queries fit where the values go");
    // (the tiles in the first 64 KB, by their alignment: an LDS instruction's own offset
    // reaches that far)
    __shared__ __align__(16384) uint8_t raw0[RAW], raw1[RAW], raw2[RAW], raw3[RAW];
    __shared__ __align__(1024) uint8_t vb[2 * kKT * PITCH];  // values in bf16 and
    __shared__ __align__(1024) uint8_t pb[2 * ROWS * 64];    // weights [row][32 keys], of tiles in turn
    // Where these two lie: a lane's place is kept with it added, as an LDS instruction's
    // own offset does not reach that far (elsewhere they would cost an addition each)
    constexpr uint32_t VB = 4 * RAW, PB = VB + 2 * kKT * PITCH;
    __shared__ uint8_t qscale[NB][ROWS];  // exponents of the queries' first pieces (255: not finite)
    __shared__ float rowred[2][ROWS];
    __shared__ uint64_t seen[ROWS];
    __shared__ uint32_t low[WIN ? ROWS : 1];
    __shared__ uint32_t bad_page, again;
    __shared__ uint64_t tmp[2 * NW + 2 + kTries / 2];
    __shared__ Req found;
    const uint32_t tid = threadIdx.x, wave = uni(tid >> 6);
    const uint32_t sr = 8u * (wave & ~1u), sk = 16u * (wave & 1u);  // first row and key of this wave's scores
    const uint32_t c = (blockIdx.x % 8u) * (kGrid / 8u) + blockIdx.x / 8u;
    const uint32_t H = p.a.n_heads, L = p.a.cache.kv_lora_rank, RP = p.a.cache.qk_rope;
    const uint32_t stride = p.a.cache.row_stride;
    if (tid == 0) bad_page = again = 0;
    const Place f = find_place<ROWS, 64 * NW, kGrid, WIN>(p, c, min_per, tmp, (u32x2*)pb, &found);
    if (tid < 2) p.desc[kDesc * (2 * c + tid)] = 0;
    Walks<ROWS, WIN> walks(p, f, c);
    auto swap = [](uint32_t row) { return 2u * (row & 7u); };
    while (walks.more()) {
        walks.find();
        const Walk w = walks.next;
        const Req& q = w.q;
        const uint32_t rt = w.rt, kt0 = w.kt0, kt1 = w.kt1, rows = walks.rows(w);
        f32x4 acc[4][CT];  // of all rows, columns 16 LC wave + [0, 16 LC)
        float m = kNone;  // the reference of row sr + n
        f32x4 l;          // the sum of row 16 (wave % 4) + n's weights, four times
        auto clear = [&]() __attribute__((always_inline)) {
            l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (uint32_t k = 0; k < CT; k++) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        };
        bool bad = false;
        if (q.flaw) {
            clear();
        } else {
            const uint32_t lane = tid & 63u, n = lane & 15u, g = lane >> 4;
            // Where the wave's rows of 64 tiles from `first_tile` on lie, one tile a lane:
            // address and bytes, found for all 64 at once, so that a turn only picks its own;
            // and the pages of the 64 behind them.
            uint32_t first_tile, t_lo, t_hi, t_size;
            int32_t more_pages;
            auto find_rows = [&](uint32_t from, int32_t page) __attribute__((always_inline)) {
                const uint32_t t = from + (afresh(tid) & 63u), key = key_of<WIN>(q, t) + DR * wave;
                const uint32_t left = t < kt1 && key < q.keys ? (q.keys - key < DR ? q.keys - key : DR) : 0u;
                const bool ok = page >= 0 && (uint32_t)page < p.a.cache.n_pages;
                bad |= left && !ok;
                const uint32_t row = ok ? ((uint32_t)page << p.psh) + (key & (p.a.cache.page_size - 1u)) : 0u;
                const uint64_t at = (uint64_t)(uintptr_t)p.a.cache.d_rows + (uint64_t)row * stride;
                first_tile = from;
                t_lo = (uint32_t)at;
                t_hi = (uint32_t)(at >> 32);
                t_size = ok && left ? (left - 1u) * stride + L / 2u + kMxScales + 2u * RP : 0u;
                more_pages = walks.page(w, t + 64u, DR * wave);
            };
            auto first_rows = [&]() __attribute__((always_inline)) {
                find_rows(kt0, walks.page(w, kt0 + (afresh(tid) & 63u), DR * wave));
            };
            // lane's chunk of the values of the wave's DR rows, of their rotary parts and scales
            const uint32_t val_i = lane >> 4, val_ch = (lane & 15u) ^ swap(DR * wave + val_i);
            const uint32_t val_at = 32u * val_ch < L ? val_i * stride + 16u * val_ch : kOOB;
            const uint32_t rot_i = (lane >> 3) & 3u, rot_ch = (lane & 7u) ^ swz8((DR * wave + rot_i) & 15u);
            // (the scales in other banks for each wave's rows)
            const uint32_t aux_at = lane >= 32u ? ((lane - 32u) / DR == wave ? (lane & 3u) * stride + L / 2u : kOOB)
                                    : 8u * rot_ch < RP ? rot_i * stride + L / 2u + kMxScales + 16u * rot_ch
                                                       : kOOB;
            auto rows_of = [&](uint32_t t) __attribute__((always_inline)) {
                if (t - first_tile >= 64u) find_rows(first_tile + 64u, more_pages);
                const int i = (int)(t - first_tile);
                const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)t_hi, i) << 32 |
                                    (uint32_t)__builtin_amdgcn_readlane((int)t_lo, i);
                return make_rsrc((const void*)at, (uint32_t)__builtin_amdgcn_readlane((int)t_size, i));
            };
            auto call_values = [&](rsrc_t rs, uint8_t* raw) __attribute__((always_inline)) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, WL_LDS(raw + 1024u * wave), 16u, val_at, 0u, 0, 0);
            };
            auto call_others = [&](rsrc_t rs, uint8_t* raw) __attribute__((always_inline)) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, WL_LDS(raw + AUX + AUXW * wave), 16u, aux_at, 0u, 0, 0);
            };
            auto call_tile = [&](uint8_t* raw, uint32_t t) __attribute__((always_inline)) {
                const rsrc_t rs = rows_of(t);
                call_values(rs, raw);
                call_others(rs, raw);
            };
            // The queries of rows sr + n: lane (row n, block g) has 32 columns of each 128 in
            // pieces, and the rotary part in bf16. They come by DMA to where the values will be,
            // 64 bytes a block; a thread cuts up a block for the two waves that need it, the
            // pieces going to the block's place and, 8 bytes of them, to the last tile's. (One
            // trip to memory, and one round of code: a walk's start takes the time that its
            // instructions take to come.) 16 bytes c of a row are at c ^ apart(row), which is
            // another place for each of 16 rows, and for the 8 rows at c and 8 at c + 4 that
            // are served together.
            auto apart = [](uint32_t row) { return 4u * ((0x1320u >> (row & 12u)) & 3u) + (row & 3u); };
            u32x6 qf[LC][QP];
            uint32_t qs[QP];  // the pieces' scales, a byte for each 128 columns
            bf16x8 qr[2];
            auto call_queries = [&]() __attribute__((always_inline)) {
                const rsrc_t ql = make_rsrc((const uint16_t*)p.a.d_q_lat + q.t0 * p.a.q_lat_stride,
                                            2u * ((q.nodes - 1u) * (uint32_t)p.a.q_lat_stride + H * L));
                const rsrc_t qro = make_rsrc((const uint16_t*)p.a.d_q_rope + q.t0 * p.a.q_rope_stride,
                                             2u * ((q.nodes - 1u) * (uint32_t)p.a.q_rope_stride + H * RP));
                // lane i has row i's place; a load brings 1 KB, of 4 / LC rows
                const uint32_t ln = afresh(tid) & 63u, row = rt * ROWS + ln, node = row / H, h = row - node * H;
                const uint32_t lat = 2u * (node * (uint32_t)p.a.q_lat_stride + h * L);
#pragma unroll 1
                for (uint32_t i = 2u * LC * wave; i < 2u * LC * (wave + 1u); i++) {
                    const uint32_t r = i * (4u / LC) + ln / (16u * LC), at = __shfl(lat, (int)r, 64);
                    const uint32_t chunk = (ln % (16u * LC)) ^ apart(r);
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(ql, WL_LDS(vb + 1024u * i), 16u,
                                                             r < rows && 8u * chunk < L ? at + 16u * chunk : kOOB, 0u, 0, 0);
                }
                const uint32_t lr = sr + (ln & 15u), mine = 2u * (node * (uint32_t)p.a.q_rope_stride + h * RP), vr = __shfl(mine, (int)lr, 64);
#pragma unroll
                for (uint32_t s = 0; s < 2; s++) {
                    const uint32_t col = 32u * s + 8u * (ln >> 4);
                    qr[s] = as_bf16x8(bld16(qro, lr < rows && col < RP ? vr + 2u * col : kOOB, 0));
                }
                if (wave == 0) {
                    uint32_t from;
                    seen[ln] = sees<WIN>(p, q, ln < rows ? node : 0u, from);
                    if (WIN) low[ln] = from;
                }
            };
            auto cut_queries = [&]() __attribute__((always_inline)) {
#pragma unroll 1
                for (uint32_t i = afresh(tid); i < ROWS * NB; i += 64u * NW) {
                    f32x16 even, odd;
                    uint32_t most = 0;
                    u32x4 x[4];
                    const uint32_t lr = i % ROWS, b = i / ROWS;
                    auto at = [&](uint32_t k) { return (u32x4*)(vb + lr * (64u * NB) + 16u * ((4u * b + k) ^ apart(lr))); };
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) x[k] = *at(k);
#pragma unroll
                    for (uint32_t k = 0; k < 16; k++) {
                        const uint32_t v = x[k / 4][k % 4];
                        even[k] = __uint_as_float(v << 16);
                        odd[k] = __uint_as_float(v & 0xFFFF0000u);
                        most = max(most, max((v << 16) & 0x7FFFFFFFu, v & 0x7FFF0000u));
                    }
                    constexpr uint32_t lo = 5u * (QP - 1u);
                    uint32_t e = (most >> 23) + ((most & 0x7FFFFFu) > 0x700000u ? 1u : 0u);
                    e = e < lo + 2u ? lo : e - 2u;
                    qscale[b][lr] = (uint8_t)(most >= 0x7F800000u ? 255u : e);
                    u32x6 y[QP];
#pragma unroll
                    for (uint32_t j = 0; j < QP; j++) {
                        const float sc = __uint_as_float((e - (j ? 5u * j - 1u : 0u)) << 23);
                        // (the conversions take several passes: their operands stay live)
                        y[j] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, sc);
                        asm volatile("" ::"v"(y[j]), "v"(even), "v"(odd), "v"(sc));
                        if (j + 1 < QP) {
                            const f32x32 z = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(y[j], sc);
                            asm volatile("" ::"v"(z), "v"(y[j]), "v"(sc));
#pragma unroll
                            for (int k = 0; k < 16; k++) {
                                even[k] -= z[2 * k];
                                odd[k] -= z[2 * k + 1];
                            }
                        }
                    }
                    *at(0) = u32x4{y[0][0], y[0][1], y[0][2], y[0][3]};
                    *at(1) = u32x4{y[0][4], y[0][5], y[1][0], y[1][1]};
                    *at(2) = u32x4{y[1][2], y[1][3], y[1][4], y[1][5]};
                    *at(3) = u32x4{y[2][0], y[2][1], y[2][2], y[2][3]};
                    *(u32x2*)(raw3 + 8u * i) = u32x2{y[2][4], y[2][5]};
                }
            };
            auto read_queries = [&]() __attribute__((always_inline)) {
                const uint32_t ln = afresh(tid) & 63u, lr = sr + (ln & 15u);
                uint32_t e = 0;
#pragma unroll
                for (uint32_t s = 0; s < LC; s++) {
                    const uint32_t b = 4u * s + (ln >> 4);
                    auto at = [&](uint32_t k) { return *(const u32x4*)(vb + lr * (64u * NB) + 16u * ((4u * b + k) ^ apart(lr))); };
                    const u32x4 x0 = at(0), x1 = at(1), x2 = at(2), x3 = at(3);
                    const u32x2 x4 = *(const u32x2*)(raw3 + 8u * (b * ROWS + lr));
                    qf[s][0] = u32x6{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1]};
                    qf[s][1] = u32x6{x1[2], x1[3], x2[0], x2[1], x2[2], x2[3]};
                    qf[s][2] = u32x6{x3[0], x3[1], x3[2], x3[3], x4[0], x4[1]};
                    e |= (uint32_t)qscale[b][lr] << (8u * s);
                }
#pragma unroll
                for (uint32_t j = 0; j < QP; j++) {
                    const uint32_t drop = (j ? 5u * j - 1u : 0u);
                    qs[j] = 0;
#pragma unroll
                    for (uint32_t s = 0; s < LC; s++) {
                        const uint32_t x = (e >> (8u * s)) & 255u;
                        qs[j] |= (x == 255u ? 255u : x - drop) << (8u * s);
                    }
                }
            };
            auto masked = [&](uint32_t t) { return is_masked<WIN>(p, q, key_of<WIN>(q, t), kKT); };
            // the key operands of step s: values of columns 128 s + 32 g of key row sk + n, or its rotary part
            const uint32_t key = sk + n, key_at = key * 256u + (16u * g ^ 16u * swap(key));
            const uint32_t key_aux = AUX + (key >> 2) * AUXW, key_rot = key_aux + (key & 3u) * 128u + 16u * (g ^ swz8(n));
            const uint32_t key_scale = key_aux + 128u * DR + 64u * (key >> 2) + (key & 3u) * 16u + 4u * g;
            // the tile's values in bf16: lane's chunk of row wave + 8 (lane / 16)
            const uint32_t cv_row = wave + 8u * (lane >> 4), cv_ch = lane & 15u;
            // (Its four pieces of 8 columns go in two pairs to the row's two halves, the pairs of
            // columns 16 k at 32 ((k / 2) + half (k % 2)): 8 lanes write to 8 places of 128 bytes,
            // with the pieces of a pair in opposite order for half of them.)
            const bool cv_odd = ((cv_ch >> 2) ^ (cv_ch >> 3)) & 1u;
            const uint32_t cv_at = cv_row * 256u + 16u * (cv_ch ^ swap(cv_row)), cv_to = cv_row * PITCH + 32u * cv_ch + (cv_odd ? 16u : 0u);
            const uint32_t cv_scale = AUX + (cv_row >> 2) * (AUXW + 64u) + 128u * DR + (cv_row & 3u) * 16u + mx_scale_at(cv_ch);
            // a tile's operands, read ahead: two steps' values, and what a lane converts
            struct Keys {
                u32x4 k[2], v;
                uint32_t scale, v_scale;
            };
            auto read_keys = [&](const uint8_t* raw, Keys& x) __attribute__((always_inline)) {
                x.scale = *(const uint32_t*)(raw + key_scale);
#pragma unroll
                for (uint32_t s = 0; s < 2; s++) x.k[s] = *(const u32x4*)(raw + (s < LC ? key_at ^ (64u * s) : key_rot));
                x.v = *(const u32x4*)(raw + cv_at);
                x.v_scale = raw[cv_scale];
            };
            // the products of rows sr + n with keys sk + 4 g + j; between them the tile's values
            // are brought to bf16 in place (VALUES), and mid(step) runs: the matrix cores run on meanwhile
            auto products = [&](const uint8_t* raw, Keys& x, f32x4& s0, uint32_t place, auto values, auto mid) __attribute__((always_inline)) {
                constexpr bool VALUES = decltype(values)::value;
                const uint32_t to = afresh(cv_to + VB) - VB + place * (kKT * PITCH), to2 = afresh((cv_to ^ 16u) + VB) - VB + place * (kKT * PITCH);
                f32x4 y[QP];
#pragma unroll
                for (uint32_t j = 0; j < QP; j++) y[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (VALUES && __ballot(x.v_scale > kMxHi)) {  // a block that is NaN: zeros (its key's scores are NaN)
                    const bool nan = x.v_scale > kMxHi;
                    x.v = nan ? u32x4{0u, 0u, 0u, 0u} : x.v;
                    x.v_scale = nan ? 0u : x.v_scale;
                }
                const float v_scale = __uint_as_float(x.v_scale << 23);
                static_for<LC>([&](auto si) __attribute__((always_inline)) {
                    constexpr int s = decltype(si)::value;
                    const u32x4 k = x.k[s % 2];
                    const i32x8 a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
#pragma unroll
                    for (uint32_t j = 0; j < QP; j++) {
                        const u32x6 b = qf[s][j];
                        const i32x8 bb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)b[4], (int)b[5], 0, 0};
                        y[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, bb, y[j], 4, 2, s, (int)x.scale, s, (int)qs[j]);
                    }
                    if (LC > 1 || s > 0) x.k[s % 2] = *(const u32x4*)(raw + (s + 2 < LC ? key_at ^ (64u * (s + 2)) : key_rot ^ (64u * (s + 2 - LC))));
                    mid(si);
                    if (VALUES && (LC == 4 || cv_ch < NB)) {
#pragma unroll
                        for (uint32_t j = 4 * s / LC; j < 4 * (s + 1) / LC; j++) {  // piece j / 2 of pair j % 2
                            const uint32_t lo = x.v[2 * (j & 1u)], hi = x.v[2 * (j & 1u) + 1u], piece = (j < 2) != cv_odd ? lo : hi;
                            *(u32x4*)(vb + (j < 2 ? to : to2) + (j & 1u) * (128u * LC)) =
                                __builtin_bit_cast(u32x4, fp4x8_bf16(piece, v_scale));
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
#pragma unroll
                for (uint32_t s = 0; s < 2; s++) {
                    if (LC == 1 && s == 1) x.k[0] = *(const u32x4*)(raw + (key_rot ^ 64u));
                    y[s] = mma(as_bf16x8(x.k[(LC + s) % 2]), qr[s], y[s]);
                }
                s0 = y[0] + (QP > 2 ? y[1] + y[QP - 1] : y[1]);
                // (255 is a NaN in the products too, 253 and 254 are not)
                const uint64_t beyond = __ballot((((x.scale & 0x7F7F7F7Fu) + 0x01010101u * (0x7Fu - kMxHi % 128u)) & x.scale & 0x80808080u) != 0u);
                if (__builtin_expect(beyond != 0u, 0)) {
                    const uint64_t keys = beyond | beyond >> 32;  // bit n: of key sk + n
                    const uint32_t nan = (uint32_t)(keys | keys >> 16) >> (4u * ((afresh(tid) & 63u) >> 4));
#pragma unroll
                    for (int k = 0; k < 4; k++) s0[k] = (nan >> k) & 1u ? __builtin_nanf("") : s0[k];
                }
            };
            // the scores in powers of two are s0 times the factor returned; those of keys
            // that the row does not see become -inf
            auto scores = [&](f32x4& s0, uint32_t t) __attribute__((always_inline)) {
                if (!masked(t)) return p.scale2;
                const uint32_t ln = afresh(tid) & 63u, lr = sr + (ln & 15u);
                const uint64_t bits = seen[lr];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t key = key_of<WIN>(q, t) + sk + 4u * (ln >> 4) + k;
                    const uint32_t bit = (uint32_t)(bits >> ((key - q.len) & 63u)) & (key < q.keys ? 1u : 0u);
                    const bool sees = key < q.len ? !WIN || key >= low[lr] || key < p.sinks : bit != 0;
                    s0[k] = sees ? s0[k] * p.scale2 : -INFINITY;
                }
                return 1.0f;
            };
            auto largest = [&](f32x4 x, float f) { return fmaxf(fmaxf(x[0] * f, x[1] * f), fmaxf(x[2] * f, x[3] * f)); };
            auto share_maxima = [&](float x) __attribute__((always_inline)) {
                const uint32_t ln = afresh(tid) & 63u, lr = sr + (ln & 15u);
                x = fmaxf(x, __shfl_xor(x, 16, 64));
                x = fmaxf(x, __shfl_xor(x, 32, 64));
                if (ln < 16u) rowred[wave & 1u][lr] = x;
                ring_barrier();
                m = fmaxf(kNone, fmaxf(rowred[0][lr], rowred[1][lr]));
            };
            auto late_maxima = [&](float x) __attribute__((always_inline)) {
                const float before = m;
                share_maxima(x);
                if (before != kNone) m = before;
            };
            bool pass = false;
            const uint32_t value_at = (4u * g + ((lane & 15u) >> 2)) * PITCH + (LC == 1 ? 32u * (wave / 2u) + 128u * (wave % 2u) : 16u * LC * wave) + 8u * (lane & 3u);
            auto vread = [&](uint32_t at, uint32_t k) __attribute__((always_inline)) {
                // columns 16 (LC wave + k): (with a single 128 columns the wave is k)
                const uint8_t* pa = vb + at + (LC == 1 ? 0u : 32u * (k / 2u) + 128u * LC * (k % 2u));
                typedef __attribute__((address_space(3))) s16x4 l_s16x4;
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa + 16 * PITCH));
                const u32x2 xx = __builtin_bit_cast(u32x2, x), yy = __builtin_bit_cast(u32x2, y);
                return u32x4{xx[0], xx[1], yy[0], yy[1]};
            };
            // chunk g of a row of weights (operand order) at g ^ turned(row): 8-byte writes meet two
            // by two, reads not at all (swz4's four by four: 49 clocks a tile more)
            const uint32_t turned = ((n & 4u) ? 3u : 0u) ^ ((n >> 1) & 1u);
            const uint32_t put_at = (sr + n) * 64u + 16u * (g ^ turned) + sk / 2u;
            const uint32_t get_at = n * 64u + 16u * (g ^ turned);
            auto put_weights = [&](f32x4 s0, float f, uint32_t place) __attribute__((always_inline)) {
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; k++) e[k] = exp2_(fmaf(s0[k], f, -m));
                *(u32x2*)(pb + (afresh(put_at + PB) - PB) + place * (ROWS * 64u)) = u32x2{pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3])};
            };
            // the values by the weights of one place; the weights' own sums are products with ones
            constexpr uint32_t VP = CT < 2 ? CT : 2;  // column tiles that the values are read ahead
            struct Values {
                bf16x8 p[4], own;
                u32x4 v[VP];
                uint32_t at;
            };
            auto read_values = [&](uint32_t place, Values& x) __attribute__((always_inline)) {
                const uint32_t get = afresh(get_at + PB) - PB + place * (ROWS * 64u);
#pragma unroll
                for (int i = 0; i < 4; i++) x.p[i] = as_bf16x8(*(const u32x4*)(pb + get + 1024u * i));
                x.own = as_bf16x8(*(const u32x4*)(pb + afresh(get_at + 1024u * (wave & 3u) + PB) - PB + place * (ROWS * 64u)));
                x.at = afresh(value_at + VB) - VB + place * (kKT * PITCH);
#pragma unroll
                for (uint32_t k = 0; k < VP; k++) x.v[k] = vread(x.at, k);
            };
            auto sums = [&](Values& x) __attribute__((always_inline)) {
                const u32x4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
#pragma unroll
                for (uint32_t v = 0; v < CT; v++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[i][v] = mma(as_bf16x8(x.v[v % VP]), x.p[i], acc[i][v]);
                    if (v + VP < CT) x.v[v % VP] = vread(x.at, v + VP);
                    if (v == 0) l = mma(as_bf16x8(ones), x.own, l);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            // A turn, between two barriers: tile t, in b1, becomes values and weights in place E,
            // tile t - 1 is summed from the other one; tile t + 3 is called for to b0, between the
            // products (at their beginning a wave stands still for it: 170 us for 163, the 64 x
            // 8). At t = kt1 the last sums.
            uint32_t fresh = kt0;  // the tile whose maxima are the references
            auto turn = [&](uint8_t* b0, const uint8_t* b1, auto place, uint32_t t) __attribute__((always_inline)) {
                constexpr uint32_t E = decltype(place)::value;
                if (t < kt1) {
                    Keys x;
                    f32x4 s0;
                    read_keys(b1, x);
                    __builtin_amdgcn_sched_barrier(0);
                    const rsrc_t rs = rows_of(t + 3);
                    products(b1, x, s0, E, std::true_type{}, [&](auto si) __attribute__((always_inline)) {
                        constexpr int s = decltype(si)::value;
                        if (s == (LC > 1 ? 1 : 0)) call_values(rs, b0);
                        if (s == LC - 1) call_others(rs, b0);
                    });
                    const float f = scores(s0, t);
                    if (t == fresh || (WIN && masked(t))) late_maxima(largest(s0, f));
                    put_weights(s0, f, E);
                }
                if (t > kt0) {
                    Values y;
                    read_values(1u - E, y);
                    __builtin_amdgcn_sched_barrier(0);
                    sums(y);
                }
                if (t >= kt1) return false;
                vm_wait<4>();  // tile t + 1 is there; t + 2 and t + 3 may be on the way
                ring_barrier();
                return true;
            };
            call_queries();
            first_rows();
            for (;;) {
                call_tile(raw0, kt0);
                call_tile(raw1, kt0 + 1);
                call_tile(raw2, kt0 + 2);
                vm_wait<0>();
                ring_barrier();
                if (fresh == kt0) {
                    cut_queries();
                    ring_barrier();
                    read_queries();
                    ring_barrier();
                }
                clear();
                for (uint32_t t = kt0;; t += 4) {
                    if (!turn(raw3, raw0, std::integral_constant<uint32_t, 0>{}, t)) break;
                    if (!turn(raw0, raw1, std::integral_constant<uint32_t, 1>{}, t + 1)) break;
                    if (!turn(raw1, raw2, std::integral_constant<uint32_t, 0>{}, t + 2)) break;
                    if (!turn(raw2, raw3, std::integral_constant<uint32_t, 1>{}, t + 3)) break;
                }
                vm_wait<0>();
                if (fresh != kt0) break;
                const uint32_t nr = afresh(tid) & 15u;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) pass |= 16u * i + nr < rows && nonfinite(acc[i]);
                pass |= l[0] > kMost;
                if (__ballot(pass) && (afresh(tid) & 63u) == 0) again = 1u;
                ring_barrier();
                const bool redo = uni(again) != 0;
                ring_barrier();
                if (!redo) break;
                if (tid == 0) again = 0u;
                float x = kNone;
                first_rows();
                for (uint32_t t = kt0; t < kt1; t++) {
                    call_tile(raw0, t);
                    vm_wait<0>();
                    ring_barrier();
                    f32x4 s0;
                    Keys y;
                    read_keys(raw0, y);
                    products(raw0, y, s0, 0, std::false_type{}, [](auto) {});
                    const float f = scores(s0, t);
                    x = fmaxf(x, largest(s0, f));
                    ring_barrier();
                }
                share_maxima(x);
                m += lift_of((kt1 - kt0) * kKT);
                ring_barrier();
                fresh = ~0u;
                first_rows();
            }
        }
        // the weights' sums over the row's lanes and waves; flaws
        const uint32_t ln = afresh(tid) & 63u, n = ln & 15u, g = ln >> 4;
        if (__ballot(bad) && ln == 0) {
            bad_page = 1u;
            set_status(p.a.d_status, WL_PAGED_E_PAGE);
        }
        if (wave < 4u && g == 0) rowred[0][16u * wave + n] = l[0];
        const bool whole = kt1 - kt0 == q.nkt;
        if (!whole && sk == 0 && g == 0) p.part_ml[2u * (w.slot * ROWS + sr + n)] = m;
        ring_barrier();
        const bool nan = bad_page != 0 || q.flaw;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lr = 16u * i + n;
            float sum = rowred[0][lr];
            if (nan) sum = __builtin_nanf("");
            if (lr < rows) {
                put_row<ROWS, LC, true, CT>(p, w, whole, lr, sum, acc[i], 16u * LC * wave + 4u * g);
                if (!whole && wave == 0 && g == 0) p.part_ml[2u * (w.slot * ROWS + lr) + 1u] = sum;
            }
        }
        if (!whole && tid == (w.slot & 1u)) walks.name_part(w);  // the thread that cleared it
        ring_barrier();
        if (tid == 0) bad_page = 0u;
        ring_barrier();
    }
}

template <int LC, bool WIN>
int run_mx4(const Tree& p, hipStream_t st) {
    hipLaunchKernelGGL((tree_mx4_kernel<LC, WIN>), dim3(kGrid), dim3(512), 0, st, p, kMinPer);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    hipLaunchKernelGGL((tree_join_kernel<kGrid, kRows16, LC, true>), dim3(2 * kGrid, 4), dim3(256), 0, st, p);
    return (int)hipGetLastError();
}

}  // namespace

int launch_tree_mx4(const wl_tree_attn& a, uint32_t window, uint32_t sinks, void* stream) {
    const Tree p = make_tree(a, window, sinks);
    hipStream_t st = (hipStream_t)stream;
    return by_class(a, [&](auto lc) {
        constexpr int LC = decltype(lc)::value;
        return window ? run_mx4<LC, true>(p, st) : run_mx4<LC, false>(p, st);
    });
}

}  // namespace paged
}  // namespace wl
