"""The paged cache in 4 bits: its rows written and read back (wl_paged_write,
wl_paged_read) and attention over them (wl_paged_tree_attention), against 64 bits."""
import numpy as np
import pytest

from windlass_amd import hip, paged

from . import paged_ref as P
from . import serving_ref as S
from .test_gpu_paged import random_trees

pytestmark = pytest.mark.gpu
i32 = lambda x: hip.DeviceBuffer.from_array(np.asarray(x, np.int32).reshape(-1))  # noqa: E731


class Write:
    """A wl_row_write into a 4-bit cache."""

    def __init__(self, seed, T, x, L, RP, H, ps, n_pages=None, pad=0, row_pad=0, slot=None, pos=None, src=None, n_kv=0, eps=2.0 ** -20,
                 kv=None, norm=None):
        rng = np.random.default_rng(seed)
        self.x, self.L, self.RP, self.H, self.T, W = x, L, RP, H, T, L + RP
        n_pages = n_pages or -(-T // ps) + 3
        self.n_pages, self.ps, self.stride = n_pages, ps, S.row_bytes(L, RP) + row_pad
        self.kv = P.as_type(rng.standard_normal((max(T, n_kv), W + pad)) if kv is None else kv, x)
        self.q = P.as_type(rng.standard_normal((T, H * RP + pad)), x)
        self.norm = P.as_type(1 + 0.1 * rng.standard_normal(L) if norm is None else norm, "bf16")
        self.pos = rng.integers(0, 1 << 20, T).astype(np.int32) if pos is None else np.asarray(pos, np.int32)
        self.slot = rng.permutation(n_pages * ps)[:T].astype(np.int32) if slot is None else np.asarray(slot, np.int32)
        self.src, self.eps, self.theta = src, eps, 1e6
        self.before = rng.integers(0, 256, (n_pages * ps, self.stride)).astype(np.uint8)
        self.cache = hip.DeviceBuffer.from_array(self.before)
        self.b = dict(d_kv=P.upload(self.kv, x), d_norm_w=P.upload(self.norm, "bf16"), d_pos=i32(self.pos), d_slot=i32(self.slot),
                      d_status=i32([0]))
        if src is not None:
            self.b["d_src"] = i32(src)
        if H:
            self.b["d_q_rope"], self.b["d_q_rope_out"] = P.upload(self.q, x), P.upload(0 * self.q, x)
        self.c = paged.Cache(d_rows=self.cache.ptr, dtype=paged.TYPE["mxfp4"], n_pages=n_pages, page_size=ps, kv_lora_rank=L,
                             qk_rope=RP, row_stride=self.stride)
        self.args = paged.RowWrite(cache=self.c, dtype=paged.TYPE[x], n_tokens=T, n_heads=H, eps=eps, rope_theta=self.theta,
                                   kv_stride=W + pad, q_stride=H * RP + pad, q_out_stride=H * RP + pad, n_kv=n_kv,
                                   **{k: v.ptr for k, v in self.b.items()})

    def run(self):
        paged.write_rows(self.args)
        hip.synchronize()
        return self

    def status(self):
        return int(self.b["d_status"].download(np.uint32)[0])

    def bytes(self):
        return self.cache.download(np.uint8).reshape(self.before.shape)

    def check(self, passed=()):
        """The compressed part's bytes are those of 64 bits (no value of these inputs is within 2^-40 of a border); rotary
        parts as paged_ref's; everything else as it was."""
        got, n = self.bytes(), S.row_bytes(self.L, self.RP)
        kept = np.ones(len(got), bool)
        for t in range(self.T):
            if t in passed or self.slot[t] < 0:
                continue
            kept[self.slot[t]] = False
            kv = self.kv[t if self.src is None else self.src[t], :self.L + self.RP]
            with np.errstate(invalid="ignore", over="ignore"):
                row = P.latent_row(kv, self.norm, self.eps, self.L, int(self.pos[t]), self.theta)
            code, e = S.quantise(row[:self.L])
            g = got[self.slot[t]]
            assert np.array_equal(g[n:], self.before[self.slot[t], n:])
            code2, e2, rope = S.unpack(g[:n], self.L)
            assert np.array_equal(e2, e)
            ok = np.repeat(e != 255, 32)
            assert np.array_equal(code2[ok], code[ok])
            used = [S.scale_at(b) for b in range(self.L // 32)]
            assert not np.delete(g[self.L // 2:self.L // 2 + 16], used).any()
            size = np.hypot(kv[self.L::2].astype(np.float64), kv[self.L + 1::2])
            far = 8 * P.U32 * np.concatenate([size, size]) * 1.01 + P.U16 * np.abs(row[self.L:]) * (1 + 1e-3)
            assert np.all(np.abs(rope - row[self.L:]) <= far)
        assert np.array_equal(got[kept], self.before[kept])
        if self.H:
            out = P.download(self.b["d_q_rope_out"], self.x, self.q.shape)[:, :self.H * self.RP].reshape(self.T, self.H, self.RP)
            q = self.q[:, :self.H * self.RP].reshape(self.T, self.H, self.RP)
            want, size = P.rope(q, self.pos[:, None], self.theta), np.hypot(q[..., 0::2].astype(np.float64), q[..., 1::2])
            u = P.U16 if self.x == "bf16" else P.U32
            far = 8.1 * P.U32 * np.concatenate([size, size], -1) + u * np.abs(want) * (1 + 1e-3)
            ok = np.abs(out - want) <= far
            ok[[t for t in passed if self.pos[t] < 0]] = True
            assert ok.all()


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("T,L,RP,H,ps,pad,row_pad", [(1, 512, 64, 64, 64, 0, 0), (1, 32, 8, 0, 8, 8, 16), (7, 96, 24, 5, 16, 16, 48),
                                                     (333, 256, 32, 20, 32, 8, 0), (1030, 480, 56, 3, 8, 0, 16), (65, 64, 64, 1, 1024, 0, 0)])
def test_write(gpu, T, L, RP, H, ps, pad, row_pad, x):
    w = Write(T + L, T, x, L, RP, H, ps, pad=pad, row_pad=row_pad).run()
    w.check()
    assert w.status() == 0


def test_write_slots_sources_and_flaws(gpu):
    w = Write(1, 4, "f32", 64, 16, 0, 16, src=[9, 0, 0, 5], n_kv=10, slot=[3, 17, -1, 0]).run()
    w.check()
    assert w.status() == 0
    w = Write(2, 7, "bf16", 64, 16, 2, 16, src=[2, 0, 3, -1, 4, 2 ** 31 - 1, -7], n_kv=4, slot=[5, 9, 0, -1, -1, -1, -1]).run()
    w.check()
    assert w.status() == 0
    w = Write(4, 6, "f32", 64, 16, 3, 16, n_pages=2, src=[0, 1, -1, 7, 3, 4], n_kv=7, slot=[32, -2, 4, 5, 6, 7],
              pos=[4, 5, 6, 7, -1, 8]).run()
    w.check(passed=(0, 1, 2, 3, 4))
    assert w.status() == paged.E_SLOT | paged.E_LEN


def test_write_values_on_borders(gpu):
    """Rows of +-1 (whose norm is 1 exactly) with weights on the borders between 4-bit values: the even code; block
    scales on theirs: the least that fits."""
    L = 128
    norm = np.array([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5] + [0.5, 1, 1.5, 2, 3, 4, 0, -0.25] + [0.2490234375, 0.251953125, 5.03125, 4.96875] +
                    [1e-30] * 12 + [6 * 2.0 ** -9] * 32 + [6.03125 * 2.0 ** 7] + [1.0] * 31 + [0.0] * 32)
    sign = np.where(np.arange(L) % 3 == 1, -1.0, 1.0)
    for x in ("f32", "bf16"):
        w = Write(5, 3, x, L, 8, 0, 8, eps=0.0, norm=norm, kv=np.concatenate([np.tile(sign * 0.125, (3, 1)), np.ones((3, 8))], 1)).run()
        w.check()
        code, e, _ = S.unpack(w.bytes()[w.slot[0]][:S.row_bytes(L, 8)], L)
        assert (code[:8] % 8).tolist() == [7, 0, 2, 2, 4, 4, 6, 6] and e.tolist() == [127, 127 - 9, 127 + 8, S.LO]
        assert not code[96:].any() and code[14] == 0 and code[15] == 0  # no negative zeros


@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_write_corners(gpu, x):
    """Rows of zeros, of the least and largest magnitudes, a NaN, an infinity; weights that are not finite spoil their own block."""
    rng = np.random.default_rng(6)
    kv = rng.standard_normal((9, 104))
    kv[0, :96] = 0
    kv[1, :96] *= 1e-36
    kv[2, :96] *= 1e36
    kv[3, 50] = np.nan
    kv[4, 3] = np.inf
    kv[5, :96] = 0
    kv[5, 17] = -1e-20
    w = Write(7, 9, x, 96, 8, 0, 8, kv=kv, eps=0.0 if x == "f32" else 2.0 ** -20)
    if x == "f32":  # 0 / 0: not finite, all blocks
        w.run().check()
        assert (S.unpack(w.bytes()[w.slot[0]][:S.row_bytes(96, 8)], 96)[1] == 255).all()
    else:
        w.run().check()
        assert (S.unpack(w.bytes()[w.slot[0]][:S.row_bytes(96, 8)], 96)[1] == S.LO).all()
    norm = np.ones(96)
    norm[40], norm[64], norm[3] = np.inf, 3.3e38, 1e-38
    w = Write(8, 4, x, 96, 8, 0, 8, norm=norm).run()
    w.check()
    e = S.unpack(w.bytes()[w.slot[0]][:S.row_bytes(96, 8)], 96)[1]
    assert e[1] == 255 and e[2] >= 250 and e[0] < 200


# ---- rows as values ------------------------------------------------------------------
def read(t, dtype, first, counts, n_rows=None, pad=0, table=None, cu=None):
    """wl_paged_read over a Serving's cache; (rows as they come back, status)."""
    cu = np.concatenate([[0], np.cumsum(counts)]) if cu is None else np.asarray(cu)
    n_rows = int(cu.max()) + 3 if n_rows is None else n_rows
    out, status = P.upload(np.full((n_rows, t.W + pad), 7.0), dtype), i32([0])
    b = dict(d_table=i32(t.table if table is None else table), d_cu=i32(cu))
    if first is not None:
        b["d_first"] = i32(first)
    paged.read_rows(paged.RowRead(cache=t.args.cache, dtype=paged.TYPE[dtype], n_req=len(t.lens), n_rows=n_rows, max_pages=t.max_pages,
                                  d_out=out.ptr, out_stride=t.W + pad, d_status=status.ptr, **{k: v.ptr for k, v in b.items()}))
    hip.synchronize()
    return P.download(out, dtype, (n_rows, t.W + pad)), int(status.download(np.uint32)[0])


@pytest.mark.parametrize("cache", ["mxfp4", "bf16", "f32"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("L,RP,ps", [(512, 64, 64), (32, 8, 8), (96, 40, 16)])
def test_read(gpu, L, RP, ps, dtype, cache):
    lens, adds = [0, 1, 63, 700, 130], [0, 0, 2, 1, 0]
    t = S.Serving(L, "f32", cache, L, RP, 2, ps, lens, adds, row_pad=16).upload()
    for first, counts in [(None, [0, 1, 65, 701, 130]), ([0, 1, 60, 333, 64], [0, 0, 5, 300, 1])]:
        got, status = read(t, dtype, first, counts, pad=8)
        assert status == 0
        want = np.concatenate([t.rows[r][(first[r] if first else 0):][:n] for r, n in enumerate(counts)])
        assert np.array_equal(got[:len(want), :t.W], P.as_type(want, dtype))  # rounded once: exact
        assert np.all(got[len(want):] == 7.0) and np.all(got[:, t.W:] == 7.0)


@pytest.mark.parametrize("cache", ["mxfp4", "bf16", "f32"])
def test_read_flaws(gpu, cache):
    t = S.Serving(9, "f32", cache, 64, 16, 2, 16, [40, 20, 33, 5], [0] * 4).upload()
    table = t.table.copy()
    table[0, 1], table[2, 0] = t.n_pages, -1
    got, status = read(t, "f32", None, [40, 20, 33, 5], table=table)
    assert status == paged.E_PAGE
    bad = np.zeros(98, bool)
    bad[16:32] = bad[60:76] = True
    want = np.concatenate(t.rows)
    assert np.isnan(got[:98][bad]).all() and np.array_equal(got[:98][~bad], want[~bad])
    for first, counts, cu, ok in [([-1, 0, 0, 0], [40, 20, 33, 5], None, [1, 2, 3]),
                                  ([0, 0, 2 ** 31 - 1, t.max_pages * 16 - 4], [40, 20, 33, 5], None, [0, 1]),
                                  (None, None, [0, 40, 60, 50, 55], [0, 1]), (None, None, [-3, 40, 60, 93, 300], [1, 2])]:
        n_rows = 101
        got, status = read(t, "f32", first, counts, n_rows=n_rows, cu=cu)
        assert status == paged.E_LEN
        at = np.concatenate([[0], np.cumsum(counts)]) if cu is None else cu
        want = np.full((n_rows, t.W), 7.0, np.float32)
        for r in ok:
            n = at[r + 1] - at[r]
            want[at[r]:at[r + 1]] = t.rows[r][:n]
        if cu == [0, 40, 60, 50, 55]:  # the last one's rows are another's too
            got, want = got[:50], want[:50]
        assert np.array_equal(got, want)


def test_read_nan_blocks(gpu):
    t = S.Serving(10, "f32", "mxfp4", 96, 16, 2, 16, [20], [0])
    page = t.table[0, 0]
    t.bytes[page, 3, 48 + S.scale_at(1)] = 255
    t.upload()
    for dtype in ("f32", "bf16"):
        got, _ = read(t, dtype, None, [20])
        want = P.as_type(t.rows[0], dtype)
        want[3, 32:64] = np.nan
        assert np.array_equal(got[:20], want, equal_nan=True)


def test_read_offsets_past_32_bits(gpu):
    for cache, size in (("mxfp4", 400), ("f32", 2304)):
        t = S.Serving(19, "f32", cache, 512, 64, 2, 64, [150], [3], first_page=(1 << 33) // (64 * size) + 1).upload()
        got, status = read(t, "bf16", None, [153])
        assert status == 0 and np.array_equal(got[:153], P.as_type(t.rows[0], "bf16"))
        t.cache.free()


# ---- attention -----------------------------------------------------------------------
Q = ["bf16", "f32"]
SHAPES = [(512, 64, 64, 64), (512, 64, 16, 16), (256, 32, 20, 32), (128, 64, 128, 64), (96, 8, 1, 8), (224, 40, 7, 8),
          (512, 64, 33, 1024), (32, 8, 3, 8), (480, 56, 9, 16), (352, 64, 2, 8)]


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("L,RP,H,ps", SHAPES)
def test_attention(gpu, L, RP, H, ps, q):
    rng = np.random.default_rng(L + H)
    lens, adds = [0, 1, 63, 130, 0, 517], [1, 3, 0, 13, 5, 2]
    t = S.Serving(L + RP + H, q, "mxfp4", L, RP, H, ps, lens, adds, random_trees(rng, adds), tail=2).upload().run()
    t.check()
    assert t.status() == 0


@pytest.mark.parametrize("q", Q)
def test_attention_chains_strides(gpu, q):
    t = S.Serving(5, q, "mxfp4", 512, 64, 8, 16, [40, 3, 300, 64], [64, 1, 9, 32], pad=24, row_pad=40, tail=1).upload().run()
    t.check()
    assert t.status() == 0


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 97, 127, 128, 129, 160, 161, 192, 193, 255, 1023])
def test_attention_one_token(gpu, q, n):
    S.Serving(n, q, "mxfp4", 512, 64, 64, 64, [n - 1], [1]).upload().run().check()


@pytest.mark.parametrize("q", Q)
def test_attention_long_and_uneven(gpu, q):
    rng = np.random.default_rng(8)
    lens, adds = [20011, 5, 700, 0, 9000], [1, 2, 64, 1, 3]
    S.Serving(9, q, "mxfp4", 512, 64, 4, 64, lens, adds, random_trees(rng, adds)).upload().run().check()


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("H,lens,adds", [(20, [900, 0, 333, 4000], [5, 1, 64, 9]), (64, list(range(0, 1200, 20)), [2] * 60),
                                         (128, [70, 2100], [64, 1])], ids=["uneven", "sixty", "tall"])
def test_attention_pieces(gpu, q, H, lens, adds):
    rng = np.random.default_rng(21)
    S.Serving(22, q, "mxfp4", 128, 32, H, 16, lens, adds, random_trees(rng, adds)).upload().run().check()


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("R", [300, 1500, 4096])
def test_attention_many_requests(gpu, q, R):
    rng = np.random.default_rng(R)
    lens, adds = [int(x) for x in rng.integers(0, 50, R)], [int(x) for x in rng.integers(0, 3, R)]
    S.Serving(24, q, "mxfp4", 64, 8, 2, 8, lens, adds, random_trees(rng, adds)).upload().run().check()


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("scale", [-0.07, 0.0])
def test_attention_scales_that_are_not_positive(gpu, q, scale):
    rng = np.random.default_rng(25)
    lens, adds = [70, 0, 611], [5, 2, 33]
    t = S.Serving(26, q, "mxfp4", 96, 16, 5, 16, lens, adds, random_trees(rng, adds))
    t.scale = scale
    t.upload().run().check()


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("power", [60, -100])
def test_attention_magnitudes(gpu, q, power):
    """Queries and rows scaled by powers of two that cancel: the same results, exact in every type."""
    t = S.Serving(27, q, "mxfp4", 128, 32, 6, 16, [300, 40], [3, 9])
    t.ql, t.qr = t.ql * np.float32(2.0 ** power), t.qr * np.float32(2.0 ** power)
    t.set_rows([x * 2.0 ** -power for x in t.rows])
    t.upload().run().check()


@pytest.mark.parametrize("q", Q)
def test_attention_queries_of_many_magnitudes(gpu, q):
    """Of the 32 queries that meet one scale a few are large: the others count by what is left of them."""
    rng = np.random.default_rng(31)
    t = S.Serving(28, q, "mxfp4", 256, 32, 6, 16, [300, 40], [3, 9])
    size = np.where(rng.random(t.ql.shape) < 0.1, 4.0, 2.0 ** rng.integers(-14, 0, t.ql.shape))
    t.ql = P.as_type(t.ql * size, q)
    t.upload().run().check()


@pytest.mark.parametrize("q", Q)
def test_attention_rows_that_see_nothing(gpu, q):
    rng = np.random.default_rng(12)
    lens, adds = [0, 70, 0, 3], [4, 4, 64, 64]
    masks = [0, 2, 0, 15] + [0, 8, 1, 0] + [int(x) for x in rng.integers(0, 1 << 62, 64)] + [0, (1 << 64) - 1] + \
        [1 << int(x) for x in rng.integers(0, 64, 62)]
    t = S.Serving(13, q, "mxfp4", 256, 64, 6, 16, lens, adds, masks).upload().run()
    t.check()
    assert np.all(t.out()[0, :6 * 256] == 0.0)


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("where", ["block", "rope"])
def test_attention_flawed_rows_reach_those_that_see_them(gpu, q, where):
    """Node 1's row has a block that is NaN, or a rotary value: its descendants are not finite, everyone else exact."""
    masks = [1, 3, 5, 11, 21, 1 << 5]
    for n in (0, 61, 200):
        t = S.Serving(14 + n, q, "mxfp4", 512, 64, 5, 32, [n, n], [6, 6], masks + masks)
        row = t.bytes[t.table[0, (n + 1) // 32], (n + 1) % 32]
        if where == "block":
            row[256 + S.scale_at(11)] = 255
        else:
            row[272 + 20:272 + 22] = [0xC0, 0x7F]
        t.upload().run()
        out = t.out()[:, :5 * 512].reshape(12, 5, 512)
        for i in range(12):
            if i in (1, 3):
                assert not np.isfinite(out[i]).all(axis=1).any()
            else:
                y, far = t.want(i // 6, i % 6)
                assert np.all(np.abs(out[i] - y) <= far)


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("k", [5, 700])
def test_attention_flawed_rows_of_the_context(gpu, q, k):
    """A block that is NaN in a row that everyone sees: everyone's results are NaN, all columns; other requests' exact."""
    t = S.Serving(33, q, "mxfp4", 256, 32, 5, 32, [900, 900], [2, 2])
    t.bytes[t.table[0, k // 32], k % 32, 128 + S.scale_at(6)] = 255
    t.upload().run().check(nan=(0,))
    assert t.status() == 0


@pytest.mark.parametrize("q", Q)
def test_attention_queries_that_are_not_finite(gpu, q):
    """They spoil their own head's row and no other."""
    for value in (np.nan, np.inf):
        t = S.Serving(34, q, "mxfp4", 128, 16, 6, 16, [100], [3])
        t.ql[1, 2 * 128 + 40] = value
        t.upload().run()
        out = t.out()[:, :6 * 128].reshape(3, 6, 128)
        assert np.isnan(out[1, 2]).all()
        for i in range(3):
            y, far = t.want(0, i) if i != 1 else (None, None)
            if y is None:
                q0, t.ql[1, 2 * 128 + 40] = t.ql[1, 2 * 128 + 40], 0
                y, far = t.want(0, 1)
                t.ql[1, 2 * 128 + 40] = q0
            ok = np.abs(out[i] - y) <= far
            assert ok[[h for h in range(6) if (i, h) != (1, 2)]].all()


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("lens,adds", [([9000], [2]), ([9000] + [1000] * 300, [2] + [1] * 300)], ids=["parts", "whole"])
def test_attention_scores_that_rise_by_more_than_a_walk_can_hold(gpu, q, lens, adds):
    """As the 16-bit cache's: scores that rise by 70 powers of two from a tile to the next, in ramps of 11 tiles."""
    t = S.Serving(36, q, "mxfp4", 128, 16, 64 if len(lens) > 1 else 256, 16, lens, adds, spread=0.5)
    n = max(lens) + max(adds)
    powers = 70.0 * (np.arange(n) % (11 * 32)) / 32
    t.qr[:, 0::16] = 128.0
    ramp = P.as_type((powers - 385) * np.log(2) / (128 * t.scale), "bf16")
    rows = t.rows
    for x in rows:
        x[:, 128] = ramp[:len(x)]
    t.set_rows(rows)
    t.upload().run().check()


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("L,H,lens,adds", [(128, 4, [40, 900], [1, 3]), (512, 64, [5000], [1]), (96, 16, [90] * 300, [1] * 300)],
                         ids=["short", "parts", "whole"])
def test_attention_values_at_the_end_of_the_range(gpu, q, L, H, lens, adds):
    """Values under the largest scale, scores of the rotary parts alone: any result lies between the values."""
    for signs in (1.0, -1.0), (1.0, 1.0):
        t = S.Serving(33, q, "mxfp4", L, 16, H, 16, lens, adds)
        rng = np.random.default_rng(34)
        t.ql[:] = 0.0
        rows = t.rows
        for x in rows:
            side = np.where(rng.random((len(x), 1)) < 0.5, signs[0], signs[1])
            x[:, :L] = side * 2.0 ** 125 * rng.choice([6.0, 4.0], (len(x), L))
        t.set_rows(rows)
        t.upload().run().check()


@pytest.mark.parametrize("q", Q)
def test_attention_refused_requests(gpu, q):
    lens, adds = [20, 30, 9, 40], [2, 3, 1, 2]

    def tree():
        return S.Serving(17, q, "mxfp4", 128, 16, 6, 16, lens, adds, tail=3)
    t = tree()
    table = t.table.copy()
    table[1, 1] = t.n_pages
    t.upload(table=table).run().check(nan=(1,))
    assert t.status() == paged.E_PAGE
    t = tree()
    t.upload(lens=[20, -5, 9, 2 ** 31 - 1]).run().check(nan=(1, 3))
    assert t.status() == paged.E_LEN
    t = tree()
    t.upload(cu=[0, 2, 5, 6, 12]).run().check(skip=(3,))
    assert t.status() == paged.E_LEN
    t = S.Serving(18, q, "mxfp4", 128, 16, 3, 16, [4, 8], [65, 2], [1] * 67).upload().run()
    t.check(nan=(0,))
    assert t.status() == paged.E_TREE


@pytest.mark.parametrize("q", Q)
def test_attention_offsets_past_32_bits(gpu, q):
    t = S.Serving(19, q, "mxfp4", 512, 64, 2, 64, [150], [3], first_page=(1 << 33) // (64 * 400) + 1)
    t.upload().run().check()
    t.cache.free()


def test_attention_most_heads(gpu):
    rng = np.random.default_rng(28)
    for q in Q:
        S.Serving(29, q, "mxfp4", 32, 8, 1024, 8, [40, 3], [2, 1], random_trees(rng, [2, 1])).upload().run().check()


@pytest.mark.parametrize("scale", [252, 253, 254])
def test_read_scales_beyond_those_of_the_write(gpu, scale):
    """253 and more count as NaN; 252 gives its values, up to 6 x 2^125."""
    t = S.Serving(11, "f32", "mxfp4", 96, 16, 2, 16, [20], [0])
    page = t.table[0, 0]
    t.bytes[page, 3, 48 + S.scale_at(1)] = scale
    t.upload()
    want = np.array(t.rows[0])
    code = t.bytes[page, 3, 16:32]
    code = np.stack([code & 15, code >> 4], 1).reshape(1, 32).astype(np.int64)
    want[3, 32:64] = S.values(code, np.array([[252]]))[0] if scale == 252 else np.nan
    for dtype in ("f32", "bf16"):
        assert np.array_equal(read(t, dtype, None, [20])[0][:20], P.as_type(want, dtype), equal_nan=True)


@pytest.mark.parametrize("q", Q)
@pytest.mark.parametrize("scale", [253, 254, 255])
@pytest.mark.parametrize("window", [0, 40])
def test_rows_of_any_bytes(gpu, q, scale, window):
    """Rows that nobody sees hold anything; the same bytes in a row that some see make their results NaN."""
    masks = [1, 3, 5, 9, 17, 33, 65, 129]  # node 1 is seen by itself alone
    n = 150
    t = S.Serving(36, q, "mxfp4", 512, 64, 4, 32, [n, n], [8, 8], masks + masks, window=window, sinks=0)
    def spoil(k):
        row = t.bytes[t.table[0, k // 32], k % 32]
        row[:256], row[256:272], row[272:] = 0x77, scale, 0x7F
    spoil(n + 1)
    if window:
        for k in range(n - window + 1):
            spoil(k)
    t.upload().run()
    out = t.out()[:, :4 * 512].reshape(16, 4, 512)
    for i in range(16):
        if i == 1:
            assert np.isnan(out[i]).all()
        else:
            y, far = t.want(i // 8, i % 8)
            assert np.all(np.abs(out[i] - y) <= far)


# ---- rows of requests of very uneven lengths -------------------------------------------
@pytest.mark.parametrize("cache,dtype", [("mxfp4", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("R", [60, 700, 4096])
def test_read_of_uneven_requests(gpu, R, cache, dtype):
    """A few long requests among many short and empty ones, most of their rows read by work-groups of other requests'."""
    rng = np.random.default_rng(R)
    lens = [int(x) for x in rng.integers(0, 4 if R < 1000 else 2, R)]
    for r, n in ((0, 2500), (R // 2, 6100), (R - 1, 3001)):
        lens[r] = n
    t = S.Serving(R, "f32", cache, 128, 16, 2, 16, lens, [0] * R).upload()
    for some in (False, True):
        first = [n // 7 for n in lens] if some else None
        counts = [n - n // 7 for n in lens] if some else lens
        got, status = read(t, dtype, first, counts, pad=8)
        assert status == 0
        want = np.concatenate([t.rows[r][(first[r] if some else 0):][:n] for r, n in enumerate(counts)])
        assert np.array_equal(got[:len(want), :t.W], P.as_type(want, dtype))
        assert np.all(got[len(want):] == 7.0) and np.all(got[:, t.W:] == 7.0)


@pytest.mark.parametrize("cache", ["mxfp4", "f32"])
def test_read_flaws_of_uneven_requests(gpu, cache):
    R = 600
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(0, 4, R)]
    lens[100], lens[400] = 6000, 5000
    t = S.Serving(6, "f32", cache, 64, 16, 2, 16, lens, [0] * R).upload()
    cu = np.concatenate([[0], np.cumsum(lens)])
    n_rows = int(cu[-1]) + 5
    want = np.full((n_rows, t.W), 7.0, np.float32)
    want[:cu[-1]] = np.concatenate(t.rows)
    table, expect = t.table.copy(), want.copy()
    table[100, 350], table[400, 0] = -1, t.n_pages  # late and early rows
    expect[cu[100] + 5600:cu[100] + 5616] = expect[cu[400]:cu[400] + 16] = np.nan
    got, status = read(t, "f32", None, lens, n_rows=n_rows, table=table)
    assert status == paged.E_PAGE and np.array_equal(got, expect, equal_nan=True)
    first = [0] * R
    first[100] = t.max_pages * 16 - 5999  # one row more than its table has
    expect = want.copy()
    expect[cu[100]:cu[101]] = 7.0
    got, status = read(t, "f32", first, lens, n_rows=n_rows)
    assert status == paged.E_LEN and np.array_equal(got, expect)
    got, status = read(t, "f32", None, lens, n_rows=int(cu[400]) + 4000)  # a long one that does not fit, and those behind it
    assert status == paged.E_LEN and np.array_equal(got, np.concatenate([want[:cu[400]], np.full((4000, t.W), 7.0)]))
    back = cu.copy()
    back[401:] -= 5000  # request 400 without rows
    back[300] = cu[300] - 6000  # it falls: request 299 is left out, 300 reads from the rows of others on
    got, status = read(t, "f32", [0] * 300 + [max(0, lens[300] - 1)] + [0] * 299, lens, n_rows=n_rows, cu=back)
    assert status == paged.E_LEN
    keep = np.ones(n_rows, bool)
    keep[back[300]:back[301]] = False  # another's too, or out of its table
    expect = want.copy()
    expect[cu[400]:] = 7.0
    expect[cu[400]:back[R]] = np.concatenate(t.rows[401:])
    expect[cu[299]:cu[300]] = 7.0
    assert np.array_equal(got[keep], expect[keep])


def test_read_of_one_long_request_among_many(gpu):
    """Its rows are read by more than the work-groups that one of many has (by those alone it takes 32 times as
    long as in a call of its own, and so 2)."""
    n, ps = 16384, 64
    cache, out = hip.DeviceBuffer(n * 1152), hip.DeviceBuffer(n * 1152)
    cache.zero()
    stream, a, b = hip.Stream(), hip.Event(), hip.Event()

    def fastest(lens):
        table = np.zeros((len(lens), n // ps), np.int32)
        table[int(np.argmax(lens))] = np.arange(n // ps)
        held = dict(d_table=i32(table), d_cu=i32(np.concatenate([[0], np.cumsum(lens)])))
        c = paged.Cache(d_rows=cache.ptr, dtype=1, n_pages=n // ps, page_size=ps, kv_lora_rank=512, qk_rope=64, row_stride=576)
        args = paged.RowRead(cache=c, dtype=1, n_req=len(lens), n_rows=n, max_pages=n // ps, d_out=out.ptr, out_stride=576,
                             **{k: v.ptr for k, v in held.items()})
        t = []
        for _ in range(12):
            a.record(stream)
            paged.read_rows(args, stream.handle)
            b.record(stream)
            b.synchronize()
            t.append(a.elapsed_ms(b))
        return min(t)
    alone = fastest([n])
    for r in (0, 200, 511):
        assert fastest([0] * r + [n] + [0] * (511 - r)) < 12 * alone
    stream.destroy()


def test_read_captured_with_other_lengths_later(gpu):
    """A captured call, replayed as the requests' lengths change: long ones come and go among many."""
    R, L, RP, ps = 500, 64, 16, 16
    lens = [20] * R
    for r in (0, 77, 250, 499):
        lens[r] = 2600
    t = S.Serving(21, "f32", "bf16", L, RP, 2, ps, lens, [0] * R).upload()
    n_rows = 8000
    out, cu = hip.DeviceBuffer(4 * n_rows * t.W), i32([0] * (R + 1))
    held = dict(d_table=i32(t.table), d_status=i32([0]))
    args = paged.RowRead(cache=t.args.cache, dtype=0, n_req=R, n_rows=n_rows, max_pages=t.max_pages, d_out=out.ptr, out_stride=t.W,
                         d_cu=cu.ptr, **{k: v.ptr for k, v in held.items()})
    stream = hip.Stream()
    g = hip.Graph(stream)
    g.begin()
    paged.read_rows(args, stream.handle)
    g.end()
    rng = np.random.default_rng(4)
    for long in ((), (77,), (0, 499), (250, 499), (), (499,)):
        counts = [int(x) for x in rng.integers(0, 5, R)]
        for r in long:
            counts[r] = int(rng.integers(1500, 2600))
        cu.upload(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        out.upload(np.full(n_rows * t.W, 7.0, np.float32))
        g.launch()
        stream.synchronize()
        got = out.download(np.float32).reshape(n_rows, t.W)
        want = np.concatenate([t.rows[r][:n] for r, n in enumerate(counts)])
        assert np.array_equal(got[:len(want)], want) and np.all(got[len(want):] == 7.0)
    assert int(held["d_status"].download(np.uint32)[0]) == 0
    stream.destroy()
