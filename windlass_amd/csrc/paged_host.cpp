// paged_host.cpp — the C ABI of the paged cache (wl_paged_*) and of the drafted
// tokens' log probabilities: checks of the argument blocks, then the launches of
// paged.hip, tree_attn.hip, tree_mx4.hip and logprobs.hip. No state but this
// thread's last message.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/windlass_moe.h"
#include "paged.h"

namespace {

thread_local char t_err[256] = "";

wl_status fail(wl_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
wl_status fail(wl_status s, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(t_err, sizeof(t_err), fmt, ap);
    va_end(ap);
    return s;
}

bool aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }
bool pow2_page(uint32_t ps) { return ps >= 8 && ps <= 1024 && (ps & (ps - 1)) == 0; }
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && na && nb && x < y + nb && y < x + na;
}
size_t esize(uint32_t t) { return t == WL_TYPE_F32 ? 4 : 2; }

// Bytes of a cache's row, of all its rows.
size_t row_bytes(const wl_paged_cache& c) {
    if (c.dtype == WL_TYPE_MXFP4) return c.kv_lora_rank / 2 + wl::paged::kMxScales + 2 * c.qk_rope;
    return (c.kv_lora_rank + c.qk_rope) * esize(c.dtype);
}
size_t cache_bytes(const wl_paged_cache& c) {
    const size_t stride = c.row_stride * (c.dtype == WL_TYPE_MXFP4 ? 1 : esize(c.dtype));
    return ((size_t)c.n_pages * c.page_size - 1) * stride + row_bytes(c);
}

wl_status check_cache(const wl_paged_cache& c) {
    if (!c.d_rows || !aligned(c.d_rows, 16)) return fail(WL_ERR_INVALID, "the cache must be 16-byte aligned and not null");
    if (c.dtype > WL_TYPE_BF16 && c.dtype != WL_TYPE_MXFP4) return fail(WL_ERR_INVALID, "cache type %u", c.dtype);
    if (!pow2_page(c.page_size)) return fail(WL_ERR_INVALID, "page_size %u: a power of two, 8 to 1024", c.page_size);
    if (c.n_pages == 0 || (uint64_t)c.n_pages * c.page_size >= (1ull << 31))
        return fail(WL_ERR_INVALID, "n_pages x page_size must be in [1, 2^31)");
    if (c.kv_lora_rank == 0 || c.kv_lora_rank % 8 || c.kv_lora_rank > 512)
        return fail(WL_ERR_INVALID, "kv_lora_rank %u: a multiple of 8, 8 to 512", c.kv_lora_rank);
    if (c.qk_rope == 0 || c.qk_rope % 8 || c.qk_rope > wl::paged::kMaxRope)
        return fail(WL_ERR_INVALID, "qk_rope %u: a multiple of 8, 8 to %u", c.qk_rope, wl::paged::kMaxRope);
    if (c.dtype == WL_TYPE_MXFP4) {
        if (c.kv_lora_rank % 32) return fail(WL_ERR_INVALID, "kv_lora_rank %u: a multiple of 32 in a 4-bit cache", c.kv_lora_rank);
        if (c.row_stride % 16 || c.row_stride < row_bytes(c) || c.row_stride > (1u << 21))
            return fail(WL_ERR_INVALID, "row_stride %u: bytes, a multiple of 16, %zu to 2^21", c.row_stride, row_bytes(c));
        return WL_OK;
    }
    if (c.row_stride % 8 || c.row_stride < c.kv_lora_rank + c.qk_rope || c.row_stride > (1u << 20))
        return fail(WL_ERR_INVALID, "row_stride %u: a multiple of 8, at least kv_lora_rank + qk_rope", c.row_stride);
    return WL_OK;
}

// A [tokens][width] array with `stride` elements from token to token.
wl_status check_rows(const void* p, uint64_t stride, uint64_t width, const char* what) {
    if (!p || !aligned(p, 16)) return fail(WL_ERR_INVALID, "%s must be 16-byte aligned and not null", what);
    if (stride % 8 || stride < width || stride > (1u << 22))
        return fail(WL_ERR_INVALID, "%s: a stride of %llu elements (a multiple of 8, %llu to 2^22)", what,
                    (unsigned long long)stride, (unsigned long long)width);
    return WL_OK;
}

// Bytes that such an array of n tokens spans.
size_t span(uint64_t stride, uint64_t width, uint64_t n, uint32_t type) {
    return n ? ((n - 1) * stride + width) * esize(type) : 0;
}

// Launches on the stream's device (a stream handle belongs to one), whatever
// the caller's current device is, which is as before afterwards.
template <class F>
wl_status on_device_of(void* stream, const char* what, F launch) {
    int cur = 0, dev = 0;
    hipError_t e = hipGetDevice(&cur);
    dev = cur;
    if (e == hipSuccess && stream) {
        hipDevice_t d = 0;
        e = hipStreamGetDevice((hipStream_t)stream, &d);
        dev = (int)d;
    }
    if (e == hipSuccess && dev != cur) e = hipSetDevice(dev);
    if (e != hipSuccess) return fail(WL_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    const int r = launch();
    if (dev != cur) (void)hipSetDevice(cur);
    if (r != 0) return fail(WL_ERR_HIP, "%s launch: %s", what, hipGetErrorString((hipError_t)r));
    return WL_OK;
}

wl_status check_tree(const wl_tree_attn* a) {
    if (!a) return fail(WL_ERR_INVALID, "the argument block is null");
    wl_status s = check_cache(a->cache);
    if (s != WL_OK) return s;
    if (a->dtype > WL_TYPE_BF16) return fail(WL_ERR_INVALID, "type %u", a->dtype);
    if (a->dtype == WL_TYPE_BF16 && a->cache.dtype == WL_TYPE_F32)
        return fail(WL_ERR_INVALID, "bf16 queries need a bf16 or 4-bit cache");
    if (a->n_req > WL_PAGED_MAX_REQ) return fail(WL_ERR_INVALID, "n_req %u exceeds %u", a->n_req, WL_PAGED_MAX_REQ);
    if (a->n_heads == 0 || a->n_heads > 1024) return fail(WL_ERR_INVALID, "n_heads %u: 1 to 1024", a->n_heads);
    if (a->n_tokens > (1u << 20)) return fail(WL_ERR_INVALID, "n_tokens %u exceeds 2^20", a->n_tokens);
    if (a->max_pages == 0 || (uint64_t)a->max_pages * a->cache.page_size >= (1ull << 31))
        return fail(WL_ERR_INVALID, "max_pages x page_size must be in [1, 2^31)");
    return WL_OK;
}

// The call through a window (0: none).
wl_status attend(const wl_tree_attn* a, uint32_t window, uint32_t sinks, const char* what, void* stream) {
    wl_status s = check_tree(a);
    if (s != WL_OK) return s;
    if (a->n_req == 0 || a->n_tokens == 0) return WL_OK;
    const wl_paged_cache& c = a->cache;
    const uint64_t H = a->n_heads, L = c.kv_lora_rank, P = c.qk_rope;
    if ((s = check_rows(a->d_q_lat, a->q_lat_stride, H * L, "d_q_lat")) != WL_OK) return s;
    if ((s = check_rows(a->d_q_rope, a->q_rope_stride, H * P, "d_q_rope")) != WL_OK) return s;
    if ((s = check_rows(a->d_out, a->out_stride, H * L, "d_out")) != WL_OK) return s;
    if (!a->d_table || !a->d_len || !a->d_cu || !aligned(a->d_table, 4) || !aligned(a->d_len, 4) || !aligned(a->d_cu, 4) ||
        !aligned(a->d_mask, 8) || !aligned(a->d_status, 4))
        return fail(WL_ERR_INVALID, "d_table, d_len and d_cu must be set and 4-byte aligned, d_mask 8-byte");
    const size_t need = wl::paged::tree_scratch(*a);
    if (!a->d_scratch || !aligned(a->d_scratch, 16) || a->scratch_bytes < need)
        return fail(WL_ERR_INVALID, "scratch of %zu bytes (%zu needed, 16-byte aligned)", a->scratch_bytes, need);
    const size_t on = span(a->out_stride, H * L, a->n_tokens, a->dtype);
    const struct {
        const void* p;
        size_t n;
    } in[] = {{a->d_q_lat, span(a->q_lat_stride, H * L, a->n_tokens, a->dtype)},
              {a->d_q_rope, span(a->q_rope_stride, H * P, a->n_tokens, a->dtype)},
              {c.d_rows, cache_bytes(c)},
              {a->d_table, 4 * (size_t)a->n_req * a->max_pages},
              {a->d_len, 4 * (size_t)a->n_req},
              {a->d_cu, 4 * ((size_t)a->n_req + 1)},
              {a->d_mask, 8 * (size_t)a->n_tokens},
              {a->d_status, 4}};
    for (const auto& x : in)
        if (overlap(a->d_out, on, x.p, x.n) || overlap(a->d_scratch, need, x.p, x.n))
            return fail(WL_ERR_INVALID, "d_out or d_scratch overlaps an input");
    if (overlap(a->d_out, on, a->d_scratch, need)) return fail(WL_ERR_INVALID, "d_scratch overlaps d_out");
    return on_device_of(stream, what, [&] { return wl::paged::launch_tree(*a, window, sinks, stream); });
}

wl_status check_logprobs(const wl_logprobs* a) {
    if (!a) return fail(WL_ERR_INVALID, "the argument block is null");
    if (a->dtype > WL_TYPE_BF16) return fail(WL_ERR_INVALID, "type %u", a->dtype);
    if (a->n_vocab == 0 || a->n_vocab > (1u << 20)) return fail(WL_ERR_INVALID, "n_vocab %u: 1 to 2^20", a->n_vocab);
    if (a->n_rows > (1u << 20) || a->n_tokens > (1u << 20)) return fail(WL_ERR_INVALID, "n_rows and n_tokens: up to 2^20");
    if (a->n_top > WL_LOGPROB_MAX_TOP || a->n_top > a->n_vocab)
        return fail(WL_ERR_INVALID, "n_top %u: up to %u and n_vocab", a->n_top, WL_LOGPROB_MAX_TOP);
    return WL_OK;
}

}  // namespace

extern "C" {

const char* wl_paged_last_error(void) { return t_err; }

wl_status wl_paged_map(const wl_page_map* m, void* stream) {
    if (!m) return fail(WL_ERR_INVALID, "the argument block is null");
    if (m->n_req > WL_PAGED_MAX_REQ) return fail(WL_ERR_INVALID, "n_req %u exceeds %u", m->n_req, WL_PAGED_MAX_REQ);
    if (!pow2_page(m->page_size)) return fail(WL_ERR_INVALID, "page_size %u: a power of two, 8 to 1024", m->page_size);
    if (m->n_pages == 0 || (uint64_t)m->n_pages * m->page_size >= (1ull << 31))
        return fail(WL_ERR_INVALID, "n_pages x page_size must be in [1, 2^31)");
    if (m->max_pages == 0 || (uint64_t)(m->n_req ? m->n_req : 1) * m->max_pages >= (1ull << 31) ||
        (uint64_t)m->max_pages * m->page_size >= (1ull << 31))
        return fail(WL_ERR_INVALID, "n_req x max_pages and max_pages x page_size must be below 2^31 (and max_pages not 0)");
    if (m->max_tokens >= (1u << 30)) return fail(WL_ERR_INVALID, "max_tokens %u exceeds 2^30", m->max_tokens);
    if (!m->d_len || !m->d_add || !m->d_have || !m->d_free || !m->d_n_free || !m->d_table || !m->d_have_out ||
        !m->d_n_free_out || !m->d_cu || (!m->d_slot && m->max_tokens))
        return fail(WL_ERR_INVALID, "only d_parent, d_pos, d_mask and d_status may be null");
    for (const void* p : {(const void*)m->d_len, (const void*)m->d_add, (const void*)m->d_have, (const void*)m->d_free,
                          (const void*)m->d_n_free, (const void*)m->d_parent, (const void*)m->d_table,
                          (const void*)m->d_have_out, (const void*)m->d_n_free_out, (const void*)m->d_cu,
                          (const void*)m->d_slot, (const void*)m->d_pos, (const void*)m->d_status})
        if (!aligned(p, 4)) return fail(WL_ERR_INVALID, "the arrays must be 4-byte aligned");
    if (!aligned(m->d_mask, 8)) return fail(WL_ERR_INVALID, "d_mask must be 8-byte aligned");
    // every work-group reads the inputs while others write the outputs
    struct Range {
        const void* p;
        size_t n;
    };
    const size_t R = m->n_req, T = m->max_tokens;
    const Range in[] = {{m->d_len, 4 * R}, {m->d_add, 4 * R}, {m->d_have, 4 * R}, {m->d_n_free, 4}, {m->d_parent, 4 * T}};
    const Range out[] = {{m->d_free, 4 * (size_t)m->n_pages}, {m->d_table, 4 * R * m->max_pages}, {m->d_have_out, 4 * R},
                         {m->d_n_free_out, 4}, {m->d_cu, 4 * (R + 1)}, {m->d_slot, 4 * T}, {m->d_pos, 4 * T},
                         {m->d_mask, 8 * T}, {m->d_status, 4}};
    const int no = (int)(sizeof(out) / sizeof(out[0]));
    for (int i = 0; i < no; i++) {
        for (const Range& x : in)
            if (overlap(out[i].p, out[i].n, x.p, x.n)) return fail(WL_ERR_INVALID, "an output overlaps an input");
        for (int j = 0; j < i; j++)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return fail(WL_ERR_INVALID, "two outputs overlap");
    }
    return on_device_of(stream, "wl_paged_map", [&] { return wl::paged::launch_map(*m, stream); });
}

wl_status wl_paged_write(const wl_row_write* w, void* stream) {
    if (!w) return fail(WL_ERR_INVALID, "the argument block is null");
    wl_status s = check_cache(w->cache);
    if (s != WL_OK) return s;
    const wl_paged_cache& c = w->cache;
    if (w->dtype > WL_TYPE_BF16) return fail(WL_ERR_INVALID, "type %u", w->dtype);
    if (w->n_heads > 1024) return fail(WL_ERR_INVALID, "n_heads %u exceeds 1024", w->n_heads);
    if (w->n_tokens > (1u << 24)) return fail(WL_ERR_INVALID, "n_tokens %u exceeds 2^24", w->n_tokens);
    if (!(w->rope_theta > 0.f) || !(w->eps >= 0.f)) return fail(WL_ERR_INVALID, "rope_theta must be positive and eps not negative");
    if (w->n_tokens == 0) return WL_OK;
    const uint32_t W = c.kv_lora_rank + c.qk_rope;
    if ((s = check_rows(w->d_kv, w->kv_stride, W, "d_kv")) != WL_OK) return s;
    if (!w->d_norm_w || !aligned(w->d_norm_w, 16)) return fail(WL_ERR_INVALID, "d_norm_w must be 16-byte aligned and not null");
    if (!w->d_pos || !w->d_slot || !aligned(w->d_pos, 4) || !aligned(w->d_slot, 4) || !aligned(w->d_src, 4) ||
        !aligned(w->d_status, 4))
        return fail(WL_ERR_INVALID, "d_pos and d_slot must be set, and index arrays 4-byte aligned");
    const size_t cache_n = cache_bytes(c);
    const size_t kv_n = span(w->kv_stride, W, w->d_src ? w->n_kv : w->n_tokens, w->dtype);
    if (overlap(c.d_rows, cache_n, w->d_kv, kv_n)) return fail(WL_ERR_INVALID, "the cache overlaps d_kv");
    if (w->n_heads) {
        const uint64_t q = (uint64_t)w->n_heads * c.qk_rope;
        if ((s = check_rows(w->d_q_rope, w->q_stride, q, "d_q_rope")) != WL_OK) return s;
        if ((s = check_rows(w->d_q_rope_out, w->q_out_stride, q, "d_q_rope_out")) != WL_OK) return s;
        const size_t qi = span(w->q_stride, q, w->n_tokens, w->dtype), qo = span(w->q_out_stride, q, w->n_tokens, w->dtype);
        const bool same = w->d_q_rope == w->d_q_rope_out && w->q_stride == w->q_out_stride;
        if (!same && overlap(w->d_q_rope, qi, w->d_q_rope_out, qo))
            return fail(WL_ERR_INVALID, "d_q_rope_out overlaps d_q_rope without being it");
        if (overlap(w->d_q_rope_out, qo, c.d_rows, cache_n) || overlap(w->d_q_rope_out, qo, w->d_kv, kv_n) ||
            overlap(w->d_q_rope, qi, c.d_rows, cache_n))
            return fail(WL_ERR_INVALID, "the rotary queries overlap the cache or d_kv");
    }
    return on_device_of(stream, "wl_paged_write", [&] { return wl::paged::launch_write(*w, stream); });
}

size_t wl_paged_tree_scratch(const wl_tree_attn* a) {
    return check_tree(a) == WL_OK ? wl::paged::tree_scratch(*a) : 0;
}

wl_status wl_paged_tree_attention(const wl_tree_attn* a, void* stream) {
    return attend(a, 0, 0, "wl_paged_tree_attention", stream);
}

wl_status wl_paged_window_attention(const wl_window_attn* w, void* stream) {
    if (!w) return fail(WL_ERR_INVALID, "the argument block is null");
    // positions are below 2^31: a longer window, or more sinks, leave out no more
    const uint32_t most = 0x7FFFFFFFu;
    return attend(&w->tree, w->window < most ? w->window : most, w->n_sinks < most ? w->n_sinks : most,
                  "wl_paged_window_attention", stream);
}

wl_status wl_paged_read(const wl_row_read* r, void* stream) {
    if (!r) return fail(WL_ERR_INVALID, "the argument block is null");
    wl_status s = check_cache(r->cache);
    if (s != WL_OK) return s;
    if (r->dtype > WL_TYPE_BF16) return fail(WL_ERR_INVALID, "type %u", r->dtype);
    if (r->n_req > WL_PAGED_MAX_REQ) return fail(WL_ERR_INVALID, "n_req %u exceeds %u", r->n_req, WL_PAGED_MAX_REQ);
    if (r->n_rows > (1u << 24)) return fail(WL_ERR_INVALID, "n_rows %u exceeds 2^24", r->n_rows);
    if (r->max_pages == 0 || (uint64_t)r->max_pages * r->cache.page_size >= (1ull << 31))
        return fail(WL_ERR_INVALID, "max_pages x page_size must be in [1, 2^31)");
    if (r->n_req == 0 || r->n_rows == 0) return WL_OK;
    const uint64_t W = r->cache.kv_lora_rank + r->cache.qk_rope;
    if ((s = check_rows(r->d_out, r->out_stride, W, "d_out")) != WL_OK) return s;
    if (!r->d_table || !r->d_cu || !aligned(r->d_table, 4) || !aligned(r->d_first, 4) || !aligned(r->d_cu, 4) ||
        !aligned(r->d_status, 4))
        return fail(WL_ERR_INVALID, "d_table and d_cu must be set, and index arrays 4-byte aligned");
    const size_t on = span(r->out_stride, W, r->n_rows, r->dtype);
    const struct {
        const void* p;
        size_t n;
    } in[] = {{r->cache.d_rows, cache_bytes(r->cache)},
              {r->d_table, 4 * (size_t)r->n_req * r->max_pages},
              {r->d_first, 4 * (size_t)r->n_req},
              {r->d_cu, 4 * ((size_t)r->n_req + 1)},
              {r->d_status, 4}};
    for (const auto& x : in)
        if (overlap(r->d_out, on, x.p, x.n)) return fail(WL_ERR_INVALID, "d_out overlaps an input");
    return on_device_of(stream, "wl_paged_read", [&] { return wl::paged::launch_read(*r, stream); });
}

size_t wl_token_logprobs_scratch(const wl_logprobs* a) {
    return check_logprobs(a) == WL_OK ? wl::paged::logprobs_scratch(*a) : 0;
}

wl_status wl_token_logprobs(const wl_logprobs* a, void* stream) {
    wl_status s = check_logprobs(a);
    if (s != WL_OK) return s;
    const size_t es = esize(a->dtype), R = a->n_rows, T = a->n_tokens, N = a->n_top;
    if (R == 0) return T == 0 ? WL_OK : fail(WL_ERR_INVALID, "tokens without rows");
    if (!a->d_logits || !aligned(a->d_logits, es)) return fail(WL_ERR_INVALID, "d_logits must be aligned to its type and not null");
    if (a->stride < a->n_vocab || a->stride > (1u << 24))
        return fail(WL_ERR_INVALID, "a stride of %llu elements (%u to 2^24)", (unsigned long long)a->stride, a->n_vocab);
    if (T && (!a->d_token || !a->d_logp)) return fail(WL_ERR_INVALID, "d_token and d_logp must be set for tokens");
    if (T > R && !a->d_row) return fail(WL_ERR_INVALID, "%u tokens of %u rows without d_row", a->n_tokens, a->n_rows);
    if (N && (!a->d_top_id || !a->d_top_logp)) return fail(WL_ERR_INVALID, "d_top_id and d_top_logp must be set for n_top");
    for (const void* p : {(const void*)a->d_token, (const void*)a->d_row, (const void*)a->d_logp, (const void*)a->d_entropy,
                          (const void*)a->d_top_logp, (const void*)a->d_top_id, (const void*)a->d_status})
        if (!aligned(p, 4)) return fail(WL_ERR_INVALID, "the arrays must be 4-byte aligned");
    const size_t need = wl::paged::logprobs_scratch(*a);
    if (!a->d_scratch || !aligned(a->d_scratch, 16) || a->scratch_bytes < need)
        return fail(WL_ERR_INVALID, "scratch of %zu bytes (%zu needed, 16-byte aligned)", a->scratch_bytes, need);
    const struct Range {
        const void* p;
        size_t n;
    } in[] = {{a->d_logits, ((R - 1) * a->stride + a->n_vocab) * es}, {a->d_token, 4 * T}, {a->d_row, 4 * T}, {a->d_status, 4}},
      out[] = {{a->d_logp, 4 * T}, {a->d_entropy, 4 * R}, {a->d_top_logp, 4 * R * N}, {a->d_top_id, 4 * R * N}, {a->d_scratch, need}};
    for (const Range& o : out) {
        for (const Range& x : in)
            if (overlap(o.p, o.n, x.p, x.n)) return fail(WL_ERR_INVALID, "an output overlaps an input");
        for (const Range& x : out)
            if (&x != &o && overlap(o.p, o.n, x.p, x.n)) return fail(WL_ERR_INVALID, "two outputs overlap");
    }
    return on_device_of(stream, "wl_token_logprobs", [&] { return wl::paged::launch_logprobs(*a, stream); });
}

}  // extern "C"
