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

// Pieces of 32 queries that meet one scale of a key: q = sum of p_i 2^s_i, p_i of E2M3;
// s_1 puts the largest into (3.75, 7.5], the others fall by 4 and 9 powers of two.
constexpr uint32_t kQueryPieces = 3;

template <int LC, bool WIN>
__global__ __launch_bounds__(512) void tree_mx4_kernel(Tree p, uint32_t min_per) {
    constexpr uint32_t NW = 8, ROWS = kRows16, PITCH = 256 * LC + kPad, CT = 2 * LC, DR = 32 / NW, QP = kQueryPieces;
    // a tile as it comes: 256 bytes of values a row, chunk c at c ^ swap(row); then by
    // wave its rows' rotary parts, chunk c at c ^ swz8(row), and scales
    constexpr uint32_t AUX = kKT * 256, AUXW = DR * 128 + 128, RAW = AUX + NW * AUXW;
    __shared__ __align__(1024) uint8_t raw0[RAW], raw1[RAW], raw2[RAW], raw3[RAW];
    __shared__ __align__(1024) uint8_t vb0[kKT * PITCH], vb1[kKT * PITCH];  // its values in bf16
    __shared__ __align__(1024) uint8_t pb0[ROWS * 64], pb1[ROWS * 64];      // weights [row][32 keys], of tiles in turn
    __shared__ float rowred[2][ROWS];
    __shared__ uint64_t seen[ROWS];
    __shared__ uint32_t low[WIN ? ROWS : 1];
    __shared__ uint32_t bad_page, again;
    __shared__ uint64_t tmp[2 * NW + 2 + kTries / 2];
    __shared__ Req found;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uni(tid >> 6), n = lane & 15u, g = lane >> 4;
    const uint32_t sr = 8u * (wave & ~1u), sk = 16u * (wave & 1u);  // first row and key of this wave's scores
    const uint32_t pr = 32u * (wave >> 2), wv = wave & 3u;          // first row of its sums, and its columns
    const uint32_t c = (blockIdx.x % 8u) * (kGrid / 8u) + blockIdx.x / 8u;
    const uint32_t H = p.a.n_heads, L = p.a.cache.kv_lora_rank, RP = p.a.cache.qk_rope;
    const uint32_t stride = p.a.cache.row_stride;
    if (tid == 0) bad_page = again = 0;
    const Place f = find_place<ROWS, 64 * NW, kGrid, WIN>(p, c, min_per, tmp, (u32x2*)pb0, &found);
    if (tid < 2) p.desc[kDesc * (2 * c + tid)] = 0;
    Walks<ROWS, WIN> walks(p, f, c);
    auto swap = [](uint32_t row) { return 2u * (row & 7u); };
    while (walks.more()) {
        walks.find();
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
        if (q.flaw) {
            clear();
        } else {
            // the pages of the wave's rows, by counted loads
            const rsrc_t table = make_rsrc(p.a.d_table + (size_t)w.r * p.a.max_pages, 4u * p.a.max_pages);
            auto page_of = [&](uint32_t t) {
                const uint32_t key = key_of<WIN>(q, t) + DR * wave, k = key < q.keys ? key : q.keys - 1u;
                return (int32_t)__builtin_amdgcn_raw_buffer_load_b32(table, (int)(4u * (k >> p.psh)), 0, 0);
            };
            // lane's chunk of the values of the wave's DR rows, of their rotary parts and scales
            const uint32_t val_i = lane >> 4, val_ch = (lane & 15u) ^ swap(DR * wave + val_i);
            const uint32_t val_at = 32u * val_ch < L ? val_i * stride + 16u * val_ch : kOOB;
            const uint32_t rot_i = (lane >> 3) & 3u, rot_ch = (lane & 7u) ^ swz8((DR * wave + rot_i) & 15u);
            const uint32_t aux_at = lane >= 32u       ? (lane & 3u) * stride + L / 2u
                                    : 8u * rot_ch < RP ? rot_i * stride + L / 2u + kMxScales + 16u * rot_ch
                                                       : kOOB;
            auto issue = [&](uint8_t* raw, uint32_t t, int32_t page_v) {
                const int32_t page = (int32_t)uni((uint32_t)page_v);
                const uint32_t key = key_of<WIN>(q, t) + DR * wave;
                const uint32_t left = t < kt1 && key < q.keys ? (q.keys - key < DR ? q.keys - key : DR) : 0u;
                const bool ok = page >= 0 && (uint32_t)page < p.a.cache.n_pages;
                bad |= left && !ok;
                const uint32_t row = ok ? ((uint32_t)page << p.psh) + (key & (p.a.cache.page_size - 1u)) : 0u;
                const rsrc_t rs = make_rsrc((const uint8_t*)p.a.cache.d_rows + (uint64_t)row * stride,
                                            ok && left ? (left - 1u) * stride + L / 2u + kMxScales + 2u * RP : 0u);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, WL_LDS(raw + 1024u * wave), 16u, val_at, 0u, 0, 0);
                if (lane < 36)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, WL_LDS(raw + AUX + AUXW * wave), 16u, aux_at, 0u, 0, 0);
            };
            // the queries of rows sr + n: lane (row n, block g) has 32 columns of each 128 in
            // pieces, and the rotary part in bf16
            u32x6 qf[LC][QP];
            uint32_t qs[QP];  // the pieces' scales, a byte for each 128 columns
            bf16x8 qr[2];
            auto read_queries = [&]() {
                const rsrc_t ql = make_rsrc((const uint16_t*)p.a.d_q_lat + q.t0 * p.a.q_lat_stride,
                                            2u * ((q.nodes - 1u) * (uint32_t)p.a.q_lat_stride + H * L));
                const rsrc_t qro = make_rsrc((const uint16_t*)p.a.d_q_rope + q.t0 * p.a.q_rope_stride,
                                             2u * ((q.nodes - 1u) * (uint32_t)p.a.q_rope_stride + H * RP));
                const uint32_t lr = sr + n, row = rt * ROWS + lr, node = row / H, h = row - node * H;
                const bool live = lr < rows;
                const uint32_t vl = 2u * (node * (uint32_t)p.a.q_lat_stride + h * L);
                const uint32_t vr = 2u * (node * (uint32_t)p.a.q_rope_stride + h * RP);
#pragma unroll
                for (uint32_t s = 0; s < 2; s++) {
                    const uint32_t col = 32u * s + 8u * g;
                    qr[s] = as_bf16x8(bld16(qro, live && col < RP ? vr + 2u * col : kOOB, 0));
                }
#pragma unroll
                for (uint32_t j = 0; j < QP; j++) qs[j] = 0;
                u32x4 x[LC][4];
#pragma unroll
                for (uint32_t s = 0; s < LC; s++) {
                    const uint32_t col = 128u * s + 32u * g;
                    const uint32_t at = live && col < L ? vl + 2u * col : kOOB;
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) x[s][k] = bld16(ql, at, 16u * k);
                }
#pragma unroll
                for (uint32_t s = 0; s < LC; s++) {
                    f32x16 even, odd;
                    uint32_t most = 0;
#pragma unroll
                    for (uint32_t k = 0; k < 16; k++) {
                        const uint32_t v = x[s][k / 4][k % 4];
                        even[k] = __uint_as_float(v << 16);
                        odd[k] = __uint_as_float(v & 0xFFFF0000u);
                        most = max(most, max((v << 16) & 0x7FFFFFFFu, v & 0x7FFF0000u));
                    }
                    constexpr uint32_t lo = 5u * (QP - 1u);
                    uint32_t e = (most >> 23) + ((most & 0x7FFFFFu) > 0x700000u ? 1u : 0u);
                    e = e < lo + 2u ? lo : e - 2u;
                    const bool nf = most >= 0x7F800000u;
#pragma unroll
                    for (uint32_t j = 0; j < QP; j++) {
                        const uint32_t ej = e - (j ? 5u * j - 1u : 0u);
                        const float sc = __uint_as_float(ej << 23);
                        // (the conversions take several passes: their operands stay live)
                        qf[s][j] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, sc);
                        asm volatile("" ::"v"(qf[s][j]), "v"(even), "v"(odd), "v"(sc));
                        qs[j] |= (nf ? 255u : ej) << (8u * s);
                        if (j + 1 < QP) {
                            const f32x32 y = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(qf[s][j], sc);
                            asm volatile("" ::"v"(y), "v"(qf[s][j]), "v"(sc));
#pragma unroll
                            for (int k = 0; k < 16; k++) {
                                even[k] -= y[2 * k];
                                odd[k] -= y[2 * k + 1];
                            }
                        }
                    }
                }
                if (sk == 0 && g == 0) {
                    uint32_t from;
                    seen[lr] = sees<WIN>(p, q, live ? node : 0u, from);
                    if (WIN) low[lr] = from;
                }
            };
            auto masked = [&](uint32_t t) { return is_masked<WIN>(p, q, key_of<WIN>(q, t), kKT); };
            // the key operands of step s: values of columns 128 s + 32 g of key row sk + n, or its rotary part
            const uint32_t key = sk + n, key_at = key * 256u + (16u * g ^ 16u * swap(key));
            const uint32_t key_aux = AUX + (key >> 2) * AUXW, key_rot = key_aux + (key & 3u) * 128u + 16u * (g ^ swz8(n));
            const uint32_t key_scale = key_aux + 128u * DR + (key & 3u) * 16u + 4u * g;
            // the products of rows sr + n with keys sk + 4 g + j
            auto products = [&](const uint8_t* raw, f32x4& s0) {
                const uint32_t ks = *(const uint32_t*)(raw + key_scale);
                u32x4 kf[LC], kr[2];
#pragma unroll
                for (uint32_t s = 0; s < LC; s++) kf[s] = *(const u32x4*)(raw + (key_at ^ (64u * s)));
#pragma unroll
                for (uint32_t s = 0; s < 2; s++) kr[s] = *(const u32x4*)(raw + (key_rot ^ (64u * s)));
                f32x4 y[QP];
#pragma unroll
                for (uint32_t j = 0; j < QP; j++) y[j] = f32x4{0.f, 0.f, 0.f, 0.f};
                static_for<LC>([&](auto si) __attribute__((always_inline)) {
                    constexpr int s = decltype(si)::value;
                    const i32x8 a = {(int)kf[s][0], (int)kf[s][1], (int)kf[s][2], (int)kf[s][3], 0, 0, 0, 0};
#pragma unroll
                    for (uint32_t j = 0; j < QP; j++) {
                        const u32x6 b = qf[s][j];
                        const i32x8 bb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)b[4], (int)b[5], 0, 0};
                        y[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, bb, y[j], 4, 2, s, (int)ks, s, (int)qs[j]);
                    }
                });
#pragma unroll
                for (uint32_t s = 0; s < 2; s++) y[s] = mma(as_bf16x8(kr[s]), qr[s], y[s]);
                s0 = y[0] + (y[1] + y[2]);
            };
            // the scores in powers of two are s0 times the factor returned; those of keys
            // that the row does not see become -inf
            auto scores = [&](f32x4& s0, uint32_t t) {
                if (!masked(t)) return p.scale2;
                const uint64_t bits = seen[sr + n];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t key = key_of<WIN>(q, t) + sk + 4u * g + k;
                    const uint32_t bit = (uint32_t)(bits >> ((key - q.len) & 63u)) & (key < q.keys ? 1u : 0u);
                    const bool sees = key < q.len ? !WIN || key >= low[sr + n] || key < p.sinks : bit != 0;
                    s0[k] = sees ? s0[k] * p.scale2 : -INFINITY;
                }
                return 1.0f;
            };
            auto largest = [&](f32x4 x, float f) { return fmaxf(fmaxf(x[0] * f, x[1] * f), fmaxf(x[2] * f, x[3] * f)); };
            auto share_maxima = [&](float x) {
                x = fmaxf(x, __shfl_xor(x, 16, 64));
                x = fmaxf(x, __shfl_xor(x, 32, 64));
                if (g == 0) rowred[wave & 1u][sr + n] = x;
                ring_barrier();
                m = fmaxf(kNone, fmaxf(rowred[0][sr + n], rowred[1][sr + n]));
            };
            auto late_maxima = [&](float x) {
                const float before = m;
                share_maxima(x);
                if (before != kNone) m = before;
            };
            bool pass = false;
            uint32_t first = kt0;  // the tile that sets the reference
            // the tile's values in bf16: lane's chunk of row wave + 8 (lane / 16)
            const uint32_t cv_row = wave + 8u * (lane >> 4), cv_ch = lane & 15u;
            auto convert = [&](const uint8_t* raw, uint8_t* vb) {
                if (LC == 4 || cv_ch < 4 * LC) {
                    const u32x4 x = *(const u32x4*)(raw + cv_row * 256u + 16u * (cv_ch ^ swap(cv_row)));
                    const uint32_t sc = raw[AUX + (cv_row >> 2) * AUXW + 128u * DR + (cv_row & 3u) * 16u + mx_scale_at(cv_ch)];
                    put_mx(x, sc, vb + cv_row * PITCH + 64u * cv_ch, cv_ch >> 2, 0u);
                }
            };
            const uint32_t value_at = (4u * g + ((lane & 15u) >> 2)) * PITCH + 64u * LC * wv + 8u * (lane & 3u);
            auto vread = [&](const uint8_t* vb, uint32_t k) {
                const uint8_t* pa = vb + value_at + 32u * k;
                typedef __attribute__((address_space(3))) s16x4 l_s16x4;
                const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa));
                const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((l_s16x4*)WL_LDS(pa + 16 * PITCH));
                const u32x2 xx = __builtin_bit_cast(u32x2, x), yy = __builtin_bit_cast(u32x2, y);
                return u32x4{xx[0], xx[1], yy[0], yy[1]};
            };
            const uint32_t put_at = (sr + n) * 64u + 16u * (g ^ swz4(n)) + sk / 2u;
            const uint32_t get_at = (pr + n) * 64u + 16u * (g ^ swz4(n));
            auto put_weights = [&](f32x4 s0, float f, uint8_t* pb) {
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; k++) e[k] = exp2_(fmaf(s0[k], f, -m));
                const u32x2 x = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3])};
                *(u32x2*)(pb + put_at) = x;
                const float r[4] = {__uint_as_float(x[0] << 16), __uint_as_float(x[0] & 0xFFFF0000u),
                                    __uint_as_float(x[1] << 16), __uint_as_float(x[1] & 0xFFFF0000u)};
                l += (r[0] + r[1]) + (r[2] + r[3]);
                pass |= fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3])) > kMost;
            };
            int32_t page0 = 0, page1 = 0;  // of the next two tiles to call for
            auto next_tile = [&](uint8_t* raw, uint32_t t) {
                const int32_t page = page0;
                page0 = page1;
                page1 = page_of(t + 2);
                issue(raw, t, page);
            };
            // between two barriers: tile t - 1 has its values in v0 and weights in w0; tile t
            // is in b1, to be brought to v1 and w1; tile t + 3's place is b0; at t = kt1 the last sums
            auto turn = [&](uint8_t* b0, const uint8_t* b1, const uint8_t* v0, uint8_t* v1, const uint8_t* w0, uint8_t* w1,
                            uint32_t t) {
                const bool live = t < kt1;
                next_tile(b0, t + 3);
                f32x4 s0;
                float f = 0.f;
                if (live) {
                    products(b1, s0);
                    f = scores(s0, t);
                    if (WIN && masked(t)) late_maxima(largest(s0, f));
                    convert(b1, v1);
                }
                bf16x8 pf[2];
#pragma unroll
                for (int i = 0; i < 2; i++) pf[i] = as_bf16x8(*(const u32x4*)(w0 + get_at + 1024u * i));
                constexpr uint32_t VP = 2;  // column tiles that the values are read ahead
                u32x4 vf[VP];
#pragma unroll
                for (uint32_t k = 0; k < VP; k++) vf[k] = vread(v0, k);
#pragma unroll
                for (uint32_t v = 0; v < CT; v++) {
#pragma unroll
                    for (int i = 0; i < 2; i++) acc[i][v] = mma(as_bf16x8(vf[v % VP]), pf[i], acc[i][v]);
                    if (v + VP < CT) vf[v % VP] = vread(v0, v + VP);
                    if (live && v == 1) put_weights(s0, f, w1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!live) return false;
                vm_wait<6>();  // tile t + 1 is there; t + 2 and t + 3 and their pages' successors may be on the way
                ring_barrier();
                return true;
            };
            for (;;) {
                clear();
                {
                    int32_t pg[5];
#pragma unroll
                    for (uint32_t i = 0; i < 5; i++) pg[i] = page_of(kt0 + i);
                    issue(raw0, kt0, pg[0]);
                    issue(raw1, kt0 + 1, pg[1]);
                    issue(raw2, kt0 + 2, pg[2]);
                    page0 = pg[3];
                    page1 = pg[4];
                }
                if (first == kt0) read_queries();
                vm_wait<0>();
                ring_barrier();
                {
                    next_tile(raw3, kt0 + 3);
                    f32x4 s0;
                    products(raw0, s0);
                    const float f = scores(s0, kt0);
                    if (first == kt0) share_maxima(largest(s0, f));
                    put_weights(s0, f, pb0);
                    convert(raw0, vb0);
                }
                ring_barrier();
                for (uint32_t t = kt0 + 1;; t += 4) {
                    if (!turn(raw0, raw1, vb0, vb1, pb0, pb1, t)) break;
                    if (!turn(raw1, raw2, vb1, vb0, pb1, pb0, t + 1)) break;
                    if (!turn(raw2, raw3, vb0, vb1, pb0, pb1, t + 2)) break;
                    if (!turn(raw3, raw0, vb1, vb0, pb1, pb0, t + 3)) break;
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
                    issue(raw0, t, page_of(t));
                    vm_wait<0>();
                    ring_barrier();
                    f32x4 s0;
                    products(raw0, s0);
                    const float f = scores(s0, t);
                    x = fmaxf(x, largest(s0, f));
                    ring_barrier();
                }
                share_maxima(x);
                m += lift_of((kt1 - kt0) * kKT);
                ring_barrier();
                first = ~0u;
            }
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
