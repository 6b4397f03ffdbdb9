"""Plain 64-bit counterparts of the 4-bit cache, the window and the log
probabilities, and the buffers of their calls, for tests/test_gpu_mx4.py,
tests/test_gpu_window.py, tests/test_gpu_logprobs.py and tests/test_gpu_serving.py."""
import numpy as np

from windlass_amd import hip, paged

from . import paged_ref as P
from .test_gpu_paged import Tree

U32, U16 = P.U32, P.U16
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LO, HI = 2, 252  # the block scales' biased exponents


# ---- rows of a 4-bit cache -------------------------------------------------------
def row_bytes(L, RP):
    return L // 2 + 16 + 2 * RP


def scale_at(b):
    return 4 * (b % 4) + b // 4


def quantise(c):
    """c [..., L] -> (codes with signs [..., L], biased exponents [..., L / 32]), by distance; blocks that are not finite
    get 255."""
    x = np.asarray(c, np.float64).reshape(*c.shape[:-1], c.shape[-1] // 32, 32)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    most = np.abs(x).max(-1)
    e = np.full(most.shape, LO - 127)
    for k in range(LO - 126, HI - 126):
        e = np.where(most > 6.0 * 2.0 ** (k - 1), k, e)
    a = np.minimum(np.abs(x) / 2.0 ** e[..., None].astype(np.float64), 6.0)
    even_first = [0, 2, 4, 6, 1, 3, 5, 7]
    code = np.array(even_first)[np.abs(a[..., None] - E2M1[even_first]).argmin(-1)]
    code = code + 8 * ((x < 0) & (code > 0))
    return code.reshape(c.shape), np.where(bad, 255, e + 127)


def values(code, exponent):
    v = np.where(code >= 8, -1.0, 1.0) * E2M1[code % 8]
    s = np.where(exponent == 255, np.nan, 2.0 ** (exponent.astype(np.float64) - 127))
    return (v.reshape(*exponent.shape, 32) * s[..., None]).reshape(code.shape)


def pack(code, exponent, rope_bits):
    """Bytes of rows [..., row_bytes] of codes [..., L], exponents and the rotary part's bf16 bits."""
    scales = np.zeros((*code.shape[:-1], 16), np.uint8)
    scales[..., [scale_at(b) for b in range(exponent.shape[-1])]] = exponent
    return np.concatenate([(code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), scales,
                           np.ascontiguousarray(rope_bits, np.uint16).view(np.uint8)], -1)


def unpack(rows, L):
    """(codes, exponents, rotary part) of bytes [..., row_bytes]."""
    n = rows[..., :L // 2].astype(np.int64)
    code = np.stack([n & 15, n >> 4], -1).reshape(*rows.shape[:-1], L)
    exponent = rows[..., L // 2:L // 2 + 16][..., [scale_at(b) for b in range(L // 32)]].astype(np.int64)
    return code, exponent, P.bf16_value(np.ascontiguousarray(rows[..., L // 2 + 16:]).view(np.uint16))


# ---- attention -------------------------------------------------------------------
def window_seen(bits, i, n, a, window, sinks):
    """What node i of a request with n tokens and a nodes sees of their n + a keys; bits: its mask."""
    seen = np.zeros(n + a, bool)
    pos = n + bin(bits & ((1 << i) - 1)).count("1")
    k = np.arange(n)
    seen[:n] = (k < sinks) | (pos - k < window) if window else True
    at = n
    for j in range(a):
        if bits >> j & 1:
            seen[n + j] = not window or at < sinks or pos - at < window
            at += 1
    return seen


def attention(q, rows, L, scale, seen, q_type, mx=False):
    """paged_ref.tree_attention_mean with what 4-bit rows add for bf16 queries: of 32 queries that meet one scale, those
    under a 120th of the largest are off by 2^-14 of it, and the products' sums by what f32 sums of the exact products
    are (their terms: three pieces of each query, at most 1.25 of it together)."""
    H = len(q)
    if not seen.any():
        return np.zeros((H, L)), np.zeros((H, L))
    q, k = q.astype(np.float64), rows[seen].astype(np.float64)
    s = scale * q @ k.T
    size = 1.25 if mx and q_type == "bf16" else 1.0
    es = (k.shape[1] * size + 16) * U32 * abs(scale) * size * (np.abs(q) @ np.abs(k).T) + 4 * U32 * np.abs(s)
    if mx and q_type == "bf16":
        b = np.abs(q[:, :L]).reshape(H, -1, 32)
        most = b.max(-1, keepdims=True)
        off = np.where((b > 0) & (b < most / 120), most * 2.0 ** -14, 0.0).reshape(H, L)
        es = es + abs(scale) * off @ np.abs(k[:, :L]).T
    es = es.max(1, keepdims=True)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    out, mag = p @ k[:, :L], p @ np.abs(k[:, :L])
    far = mag * np.expm1(2 * es + (len(k) + 80) * U32)
    if q_type == "bf16":
        dev = np.stack([w @ np.abs(k[:, :L] - o) for w, o in zip(p, out)])
        far = (far + U16 / (1 - U16) * dev) * (1 + U16) + U16 * np.abs(out)
    return out, far + 1e-37


class Serving(Tree):
    """A Tree over any cache ("mxfp4" too), through a window or not (0)."""

    def __init__(self, seed, q, cache, L, RP, H, ps, lens, adds, masks=None, window=0, sinks=0, **more):
        super().__init__(seed, q, "f32" if cache == "mxfp4" else cache, L, RP, H, ps, lens, adds, masks, **more)
        self.window, self.sinks, self.mx = window, sinks, cache == "mxfp4"
        if self.mx:
            self.set_rows([r.astype(np.float64) for r in self.rows])

    def set_rows(self, rows):
        """Values (finite) for the requests' rows, as a 4-bit cache holds them."""
        small, RP = self.pages.shape[0], self.W - self.L
        self.byte_stride = row_bytes(self.L, RP) + 16 * ((self.stride - self.W) // 8)
        self.bytes = np.full((small, self.ps, self.byte_stride), 0xFF, np.uint8)  # rows that belong to nobody: NaN
        self.rows = []
        for r, x in enumerate(rows):
            code, e = quantise(x[:, :self.L])
            bits = P.bf16_bits(x[:, self.L:])
            self.rows.append(np.concatenate([values(code, e), P.bf16_value(bits)], 1))
            b = pack(code, e, bits)
            for k in range(len(x)):
                self.bytes[self.table[r, k // self.ps] - self.first_page, k % self.ps, :b.shape[1]] = b[k]

    def spoil(self, r, k):
        """Makes row k of request r NaN."""
        page = self.table[r, k // self.ps] - self.first_page
        if self.mx:
            self.bytes[page, k % self.ps] = 0xFF
        else:
            self.pages[page, k % self.ps] = np.nan

    def upload(self, **change):
        if not self.mx:
            return super().upload(**change)
        self.ct, pages = "bf16", self.pages
        self.pages = self.pages[:0]
        super().upload(**change)  # (the buffers but the cache's)
        self.ct, self.pages = "mxfp4", pages
        self.cache.free()
        n = self.ps * self.byte_stride
        self.cache = hip.DeviceBuffer(self.n_pages * n)
        self.cache.upload(self.bytes, self.first_page * n)
        c = self.args.cache
        c.d_rows, c.dtype, c.row_stride = self.cache.ptr, paged.TYPE["mxfp4"], self.byte_stride
        assert paged.tree_attention_scratch(self.args) == self.args.scratch_bytes
        return self

    def call(self, stream=0):
        if self.window:
            paged.window_attention(paged.WindowAttention(tree=self.args, window=self.window, n_sinks=self.sinks), stream)
        else:
            paged.tree_attention(self.args, stream)

    def run(self, stream=0):
        self.call(stream)
        hip.synchronize()
        return self

    def seen(self, r, i):
        t = self.cu[r] + i
        bits = (2 << i) - 1 if self.masks is None else int(self.masks[t])
        return window_seen(bits, i, self.lens[r], self.adds[r], self.window, self.sinks)

    def want(self, r, i):
        t = self.cu[r] + i
        q = np.concatenate([self.ql[t, :self.H * self.L].reshape(self.H, self.L),
                            self.qr[t, :self.H * (self.W - self.L)].reshape(self.H, -1)], 1)
        return attention(q, self.rows[r], self.L, self.scale, self.seen(r, i), self.qt, self.mx)


# ---- log probabilities -------------------------------------------------------------
def logprobs(z):
    """Of rows z in 64 bits: (log p, entropy, how far log p may be off without its own logit's part, how far the entropy).

    With u = 2^-24 and d = z - M: an exponential is off by 4 u |d| + 3 u relatively (the difference, the product with
    log2 e twice, the exponential's own), brought to new references by as much again in all; a lane adds len / 64
    values one by one (fewer where a row has parts), its sums are rescaled once for each 2048, and joined a hundred
    times at the most. Logarithm, difference and quotient: 8 u of their results."""
    z = np.asarray(z, np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = z.max(-1, keepdims=True)
        d = z - m
        e = np.exp(d)
        s = e.sum(-1, keepdims=True)
        p = e / s
        dz = np.where(e > 0, d, 0.0)
        mean, square = (p * -dz).sum(-1), (p * dz * dz).sum(-1)
        log_s = np.log(s)[..., 0]
        rel = (z.shape[-1] / 64 * (1 + 4 / 32) + 500 + 8 * mean) * U32
        logp = d - log_s[..., None]
        far = rel + 8 * U32 * np.abs(log_s)
        entropy = log_s + mean
        far_e = far + rel * mean + 16 * U32 * (square + mean + np.abs(entropy))
    return logp, entropy, far, far_e


def order(z, n):
    """Ids of the n largest: descending, NaN first, equal ones (zeros of either sign too) by id."""
    key = np.where(np.isnan(z), np.inf, np.asarray(z, np.float64))
    return np.lexsort((np.arange(len(z)), -key, ~np.isnan(z)))[:n]


class Logprobs:
    """The buffers of a wl_logprobs. off: elements that d_logits lies behind an aligned address."""

    def __init__(self, z, t, token, row=None, n_top=0, pad=0, off=0, entropy=True, fill=9.0):
        R, V = z.shape
        self.z, self.t, self.token, self.row, self.n_top, self.fill = P.as_type(z, t), t, token, row, n_top, fill
        stride = V + pad
        flat = np.full(off + R * stride, fill, np.float32)
        flat[off:].reshape(R, stride)[:, :V] = self.z
        i32 = lambda x: hip.DeviceBuffer.from_array(np.asarray(x, np.int32).reshape(-1))  # noqa: E731
        f32 = lambda n: hip.DeviceBuffer.from_array(np.full(n, fill, np.float32))  # noqa: E731
        self.logits = P.upload(flat, t)
        T = len(token)
        self.b = dict(d_status=i32([0]))
        if T:
            self.b.update(d_token=i32(token), d_logp=f32(T + 1))
        if row is not None:
            self.b["d_row"] = i32(row)
        if entropy:
            self.b["d_entropy"] = f32(R + 1)
        if n_top:
            self.b.update(d_top_logp=f32(R * n_top + 1), d_top_id=i32([-5] * (R * n_top + 1)))
        self.args = paged.TokenLogprobs(dtype=paged.TYPE[t], n_rows=R, n_vocab=V, n_tokens=T, n_top=n_top,
                                        d_logits=self.logits.ptr + off * (2 if t == "bf16" else 4), stride=stride,
                                        **{k: v.ptr for k, v in self.b.items()})
        n = paged.token_logprobs_scratch(self.args)
        self.b["d_scratch"] = hip.DeviceBuffer.from_array(np.full(n, 0xFF, np.uint8))
        self.args.d_scratch, self.args.scratch_bytes = self.b["d_scratch"].ptr, n

    def run(self, stream=0):
        paged.token_logprobs(self.args, stream)
        hip.synchronize()
        return self

    def get(self, name, n, t=np.float32):
        x = self.b["d_" + name].download(t, n + 1)
        assert x[n] == (-5 if t == np.int32 else self.fill)  # what nobody writes
        return x[:n]

    def status(self):
        return int(self.b["d_status"].download(np.uint32)[0])

    def check(self, bad_tokens=()):
        R, V = self.z.shape
        logp, entropy, far, far_e = logprobs(self.z)
        live = np.isfinite(entropy)  # rows without a finite logit, with a NaN or +infinity: NaN
        def near(got, want, tol):
            with np.errstate(invalid="ignore"):
                ok = (np.abs(got - want) <= tol + 8 * U32 * np.abs(want)) | (got == want)
            assert ok.all(), (got[~ok][:4], want[~ok][:4])
        if len(self.token):
            got = self.get("logp", len(self.token))
            row = np.arange(len(self.token)) if self.row is None else np.asarray(self.row)
            for i, (r, k) in enumerate(zip(row, self.token)):
                if i in bad_tokens or not live[r]:
                    assert np.isnan(got[i])
                else:
                    near(got[i:i + 1], logp[r, k:k + 1], far[r])
        if "d_entropy" in self.b:
            got = self.get("entropy", R)
            assert np.isnan(got[~live]).all()
            near(got[live], entropy[live], far_e[live])
        if self.n_top:
            ids = self.get("top_id", R * self.n_top, np.int32).reshape(R, -1)
            got = self.get("top_logp", R * self.n_top).reshape(R, -1)
            for r in range(R):
                want = order(self.z[r], self.n_top)
                assert np.array_equal(ids[r], want), (r, ids[r], want)
                if live[r]:
                    near(got[r], logp[r, want], far[r])
                else:
                    assert np.isnan(got[r]).all()
