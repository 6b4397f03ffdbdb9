"""The page map, the write of latent rows and tree attention against plain
64-bit counterparts (tests/paged_ref.py), at the sizes, masks and flaws where
they can go wrong."""
import numpy as np
import pytest

from tests import paged_ref as P
from windlass_amd import hip, paged

pytestmark = pytest.mark.gpu


# ---- the page map -----------------------------------------------------------
def make_step(rng, R, ps, max_add, max_len, trees):
    lens = [int(x) for x in rng.integers(0, max_len + 1, R)]
    adds = [int(x) for x in rng.integers(0, max_add + 1, R)]
    if R > 2:
        lens[1], adds[1] = 0, 0  # an ended request
        adds[0] = max_add
    have = [-(-n // ps) + int(rng.integers(0, 4)) for n in lens]
    max_pages = max(have + [-(-(n + a) // ps) for n, a in zip(lens, adds)]) + 1
    new = sum(max(0, -(-(n + a) // ps) - h) for n, a, h in zip(lens, adds, have))
    n_free = max(0, new - sum(max(0, h - -(-(n + a) // ps)) for n, a, h in zip(lens, adds, have))) + 2
    n_pages = sum(have) + n_free + 5
    pages = rng.permutation(n_pages).astype(np.int32)
    table = np.full((R, max_pages), -9, np.int32)
    at = n_free
    for r, h in enumerate(have):
        table[r, :h] = pages[at:at + h]
        at += h
    free = np.full(n_pages, -5, np.int32)
    free[:n_free] = pages[:n_free]
    parent = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(a)] for a in adds] + [[]]).astype(np.int32) \
        if trees else None
    return dict(ps=ps, n_pages=n_pages, max_pages=max_pages, lens=lens, adds=adds, have=have, free=free, n_free=n_free,
                table=table, parent=parent)


def check_step(m, s, extra=0):
    table, free, have, n_free, cu, slot, pos, mask = P.page_map(s["ps"], s["max_pages"], s["n_pages"], s["lens"], s["adds"],
                                                                s["have"], s["free"], s["n_free"], s["table"], s["parent"])
    n = len(slot)
    assert m.get("status")[0] == 0
    assert np.array_equal(m.get("table"), table)
    assert np.array_equal(m.get("free"), free)
    assert np.array_equal(m.get("have_out"), have) and m.get("n_free_out")[0] == n_free
    assert np.array_equal(m.get("cu"), cu)
    assert np.array_equal(m.get("slot")[:n], slot) and np.array_equal(m.get("pos")[:n], pos)
    if "d_mask" in m.b:
        assert np.array_equal(m.get("mask")[:n], np.array(mask, np.uint64))
        assert np.all(m.get("mask")[n:] == 77)
    assert np.all(m.get("slot")[n:] == -1) and np.all(m.get("pos")[n:] == 0)  # behind the last request: no tokens


@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("R,ps,max_add,max_len", [(1, 8, 1, 0), (1, 16, 64, 40), (3, 8, 5, 9), (37, 16, 64, 300),
                                                  (256, 64, 64, 2000), (257, 32, 33, 500), (1024, 8, 9, 200),
                                                  (1025, 16, 17, 100), (4096, 128, 6, 700)])
def test_map(gpu, R, ps, max_add, max_len, trees):
    s = make_step(np.random.default_rng(R + ps), R, ps, max_add, max_len, trees)
    m = P.Map(**s, max_tokens=sum(s["adds"]) + 3)
    for _ in range(2):  # again on the same buffers: the same outputs
        paged.page_map(m.args)
        hip.synchronize()
        check_step(m, s)


def test_map_long_prompts_and_chain_masks(gpu):
    s = make_step(np.random.default_rng(2), 9, 16, 3001, 5000, False)
    m = P.Map(**s)
    paged.page_map(m.args)
    hip.synchronize()
    check_step(m, s)
    s = make_step(np.random.default_rng(3), 9, 16, 64, 5000, False)
    m = P.Map(**s, trees=True)  # masks without parents: chains
    paged.page_map(m.args)
    hip.synchronize()
    check_step(m, s)


@pytest.mark.parametrize("shift", [0, 4])
def test_map_long_runs(gpu, shift):
    """More than 2^18 tokens, where a thread takes four: ends of requests inside the four,
    requests of one and of no token, pages outside the cache, outputs that are not 16-byte aligned."""
    adds = [70001, 0, 1, 0, 3, 130002, 64, 1, 2, 90000]
    lens = [13, 40, 0, 16, 15, 31, 4096, 0, 7, 50]
    have = [-(-n // 16) for n in lens]
    need = [-(-(n + a) // 16) for n, a in zip(lens, adds)]
    n_free = sum(need) - sum(have)
    n_pages = sum(need) + 4
    rng = np.random.default_rng(5)
    pages = rng.permutation(n_pages).astype(np.int32)
    table = np.full((10, max(need)), -9, np.int32)
    at = n_free
    for r, h in enumerate(have):
        table[r, :h] = pages[at:at + h]
        at += h
    free = np.full(n_pages, -5, np.int32)
    free[:n_free] = pages[:n_free]
    free[n_free - 3] = n_pages  # the third page taken
    s = dict(ps=16, n_pages=n_pages, max_pages=max(need), lens=lens, adds=adds, have=have, free=free, n_free=n_free,
             table=table, parent=None)
    m = P.Map(**s, max_tokens=sum(adds) + 7)
    m.args.max_tokens -= shift // 4
    m.args.d_slot += shift
    m.args.d_pos += shift
    paged.page_map(m.args)
    hip.synchronize()
    want = P.page_map(16, s["max_pages"], n_pages, lens, adds, have, free, n_free, table)
    slot, n, o = want[5], sum(adds), shift // 4
    slot[slot >= n_pages * 16] = -1
    assert m.get("status")[0] == paged.E_PAGE
    assert np.array_equal(m.get("table"), want[0]) and np.array_equal(m.get("cu"), want[4])
    assert np.count_nonzero(slot == -1) == 16
    assert np.array_equal(m.get("slot")[o:o + n], slot) and np.array_equal(m.get("pos")[o:o + n], want[6])
    for x, none in (m.get("slot"), -1), (m.get("pos"), 0):
        assert np.all(x[:o] == -7) and np.all(x[o + n:] == none)


@pytest.mark.parametrize("trees", [False, True])
def test_map_and_write_with_room_for_more(gpu, trees):
    """Buffers for 40 tokens: a step of 30, then one of 3. Its write leaves the rows of the first alone."""
    L, RP, ps, n_pages = 32, 8, 8, 12
    W = L + RP
    rng = np.random.default_rng(31)
    parent = np.full(40, -1, np.int32) if trees else None
    m = P.Map(ps, n_pages, 6, [0, 0], [10, 20], [0, 0], np.arange(n_pages), n_pages, np.full((2, 6), -1), parent, max_tokens=40)
    norm = P.as_type(np.ones(L), "bf16")
    b = dict(d_kv=P.upload(rng.standard_normal((40, W)), "f32"), d_norm_w=P.upload(norm, "bf16"),
             cache=P.upload(np.zeros((n_pages * ps, W)), "f32"))
    c = paged.Cache(d_rows=b["cache"].ptr, dtype=paged.TYPE["f32"], n_pages=n_pages, page_size=ps, kv_lora_rank=L, qk_rope=RP,
                    row_stride=W)
    w = paged.RowWrite(cache=c, dtype=paged.TYPE["f32"], n_tokens=40, eps=1e-6, rope_theta=1e4, kv_stride=W, d_kv=b["d_kv"].ptr,
                       d_norm_w=b["d_norm_w"].ptr, d_pos=m.b["d_pos"].ptr, d_slot=m.b["d_slot"].ptr,
                       d_status=m.b["d_status"].ptr)
    kept = None
    for lens, adds in ([0, 0], [10, 20]), ([10, 20], [1, 2]):
        m.b["d_len"].upload(np.asarray(lens, np.int32))
        m.b["d_add"].upload(np.asarray(adds, np.int32))
        if kept is not None:
            m.b["d_have"].upload(m.get("have_out").astype(np.int32))
            m.b["d_n_free"].upload(m.get("n_free_out").astype(np.int32))
            b["d_kv"].upload(rng.standard_normal((40, W)).astype(np.float32))
        paged.page_map(m.args)
        paged.write_rows(w)
        hip.synchronize()
        assert m.get("status")[0] == 0
        slots, rows = m.get("slot"), P.download(b["cache"], "f32", (n_pages * ps, W))
        n = sum(adds)
        assert np.all(slots[:n] >= 0) and np.all(slots[n:] == -1)
        if kept is not None:
            still = np.setdiff1d(np.arange(n_pages * ps), slots[:n])
            assert np.array_equal(rows[still], kept[still])
            assert not np.any(np.all(rows[slots[:n]] == kept[slots[:n]], axis=1))
        kept = rows


def test_map_many_pages_given_back(gpu):
    """Ended requests' pages, far more of them than tokens."""
    R, held = 40, 900
    lens, adds = [0 if r % 3 else 100 + r for r in range(R)], [0 if r % 3 else 1 for r in range(R)]
    have = [held - 7 * r for r in range(R)]
    n_pages = sum(have) + 3
    pages = np.random.default_rng(6).permutation(n_pages).astype(np.int32)
    table, at = np.full((R, held), -9, np.int32), 3
    for r, h in enumerate(have):
        table[r, :h] = pages[at:at + h]
        at += h
    free = np.full(n_pages, -5, np.int32)
    free[:3] = pages[:3]
    s = dict(ps=8, n_pages=n_pages, max_pages=held, lens=lens, adds=adds, have=have, free=free, n_free=3, table=table,
             parent=None)
    m = P.Map(**s)
    paged.page_map(m.args)
    hip.synchronize()
    check_step(m, s)


def test_map_no_requests(gpu):
    m = P.Map(16, 4, 1, [], [], [], [0, 1, 2, 3], 4, np.zeros((0, 1), np.int32), max_tokens=2)
    paged.page_map(m.args)
    hip.synchronize()
    assert m.get("cu")[0] == 0 and m.get("n_free_out")[0] == 4 and m.get("status")[0] == 0


def test_map_takes_pages_it_pushes(gpu):
    """An empty stack: the growing request's pages are the ended ones', the last pushed first."""
    table = np.array([[3, 1, 2, -1], [0, -1, -1, -1], [5, 4, -1, -1]], np.int32)
    s = dict(ps=8, n_pages=6, max_pages=4, lens=[0, 7, 0], adds=[0, 24, 0], have=[3, 1, 2], free=np.full(6, -5, np.int32),
             n_free=0, table=table, parent=None)
    m = P.Map(**s)
    paged.page_map(m.args)
    hip.synchronize()
    check_step(m, s)
    assert m.get("table")[1].tolist() == [0, 4, 5, 2]


REFUSED = [("negative length", dict(lens=[10, -1, 0]), paged.E_LEN),
           ("negative addition", dict(adds=[4, -2, 1]), paged.E_LEN),
           ("pages missing for the tokens held", dict(have=[1, 0, 0]), paged.E_LEN),
           ("more pages than the table's row", dict(have=[1, 9, 0]), paged.E_LEN),
           ("a request longer than its row", dict(adds=[4, 2 ** 31 - 1, 1]), paged.E_LEN),
           ("more tokens than the arrays hold", dict(max_tokens=14), paged.E_LEN),
           ("a stack above the cache", dict(n_free=9), paged.E_PAGE),
           ("a stack below nothing", dict(n_free=-1), paged.E_PAGE),
           ("too few pages", dict(n_free=1), paged.E_SPACE)]


@pytest.mark.parametrize("what,change,bit", REFUSED, ids=[x[0] for x in REFUSED])
def test_map_refused_on_the_device(gpu, what, change, bit):
    table = np.array([[3, 1, -1], [0, -1, -1], [-1, -1, -1]], np.int32)
    s = dict(ps=8, n_pages=8, max_pages=3, lens=[10, 8, 0], adds=[4, 10, 1], have=[2, 1, 0],
             free=np.array([2, 4, 5, 6, 7, -5, -5, -5], np.int32), n_free=5, table=table, parent=None)
    s = {**s, **change}
    m = P.Map(**{"max_tokens": 15, **s})
    paged.page_map(m.args)
    hip.synchronize()
    assert m.get("status")[0] == bit
    assert np.all(m.get("cu") == 0) and np.all(m.get("slot") == -1)
    assert m.get("have_out").tolist() == s["have"] and m.get("n_free_out")[0] == s["n_free"]
    assert np.array_equal(m.get("table"), table) and np.array_equal(m.get("free"), s["free"]) and np.all(m.get("pos") == -7)


def test_map_too_large_trees_and_wrong_parents(gpu):
    base = dict(ps=64, n_pages=4, max_pages=2, lens=[0], have=[0], free=np.arange(4, dtype=np.int32), n_free=4,
                table=np.full((1, 2), -1, np.int32))
    m = P.Map(**base, adds=[65], parent=np.arange(65) - 1)
    paged.page_map(m.args)
    hip.synchronize()
    assert m.get("status")[0] == paged.E_TREE and np.all(m.get("slot") == -1)
    parent = np.array([-1, 0, 2, -2, 9, 1], np.int32)  # node 2 its own, -2, a later one: each counts as -1
    s = dict(base, adds=[6], parent=parent)
    m = P.Map(**s)
    paged.page_map(m.args)
    hip.synchronize()
    assert m.get("status")[0] == paged.E_TREE
    assert m.get("mask").tolist() == P.page_map(64, 2, 4, [0], [6], [0], s["free"], 4, s["table"], parent)[7]
    assert m.get("pos").tolist() == [0, 1, 0, 0, 0, 2]


def test_map_pages_outside_the_cache(gpu):
    s = dict(ps=8, n_pages=6, max_pages=3, lens=[6, 7], adds=[1, 3], have=[1, 1], n_free=2, parent=None,
             free=np.array([99, -3, 0, 0, 0, 0], np.int32), table=np.array([[6, -1, -1], [1, -1, -1]], np.int32))
    m = P.Map(**s)
    paged.page_map(m.args)
    hip.synchronize()
    assert m.get("status")[0] == paged.E_PAGE
    assert m.get("slot").tolist() == [-1, 15, -1, -1]  # a held page, a held one, and a taken one


@pytest.mark.parametrize("flaw", [-1, 6, 2 ** 31 - 1])
@pytest.mark.parametrize("trees", [False, True])
def test_map_gives_back_pages_outside_the_cache(gpu, flaw, trees):
    """Entries of an ended request that are no pages, with nobody who takes them in this step: they are found where
    they are given back, not when another request is served with them."""
    s = dict(ps=8, n_pages=6, max_pages=3, lens=[0, 7], adds=[0, 1], have=[3, 1], n_free=1, parent=np.array([-1]) if trees else None,
             free=np.array([5, 0, 0, 0, 0, 0], np.int32), table=np.array([[2, flaw, 3], [1, -1, -1]], np.int32))
    m = P.Map(**s)
    paged.page_map(m.args)
    hip.synchronize()
    assert m.get("status")[0] == paged.E_PAGE
    assert m.get("slot").tolist() == [15] and m.get("have_out").tolist() == [0, 1]
    assert m.get("n_free_out")[0] == 4 and m.get("free")[:4].tolist() == [5, 2, flaw, 3]  # counts and order as always


# ---- the write ----------------------------------------------------------------
class Write:
    def __init__(self, seed, T, x, cache, L, RP, H, ps, pad=0, pos=None, slot=None, n_pages=None, src=None, n_kv=None,
                 in_place=False, status=True):
        rng = np.random.default_rng(seed)
        W = L + RP
        self.T, self.x, self.ct, self.L, self.RP, self.H, self.W = T, x, cache, L, RP, H, W
        n_kv = T if n_kv is None else n_kv
        n_pages = -(-T // ps) + 2 if n_pages is None else n_pages
        self.n_kv, self.rows, self.stride = n_kv, n_pages * ps, W + 2 * pad
        self.ks, self.qs, self.os = W + pad, H * RP + pad, H * RP + (pad if in_place else 3 * pad)
        self.kv = P.as_type(rng.standard_normal((n_kv, self.ks)), x)
        self.q = P.as_type(rng.standard_normal((T, self.qs)), x)
        self.w = P.as_type(1 + 0.1 * rng.standard_normal(L), "bf16")
        self.pos = rng.integers(0, 1 << 20, T).astype(np.int32) if pos is None else np.asarray(pos, np.int32)
        self.slot = rng.permutation(self.rows)[:T].astype(np.int32) if slot is None else np.asarray(slot, np.int32)
        self.src = None if src is None else np.asarray(src, np.int32)
        self.theta, self.eps = 1e6, 1e-6
        self.b = dict(d_kv=P.upload(self.kv, x), d_norm_w=P.upload(self.w, "bf16"),
                      d_pos=hip.DeviceBuffer.from_array(self.pos), d_slot=hip.DeviceBuffer.from_array(self.slot))
        self.rows0 = P.as_type(np.full((self.rows, self.stride), 3.0), cache)
        self.cache = P.upload(self.rows0, cache)
        if src is not None:
            self.b["d_src"] = hip.DeviceBuffer.from_array(self.src)
        if H:
            self.b["d_q_rope"] = P.upload(self.q, x)
            self.b["d_q_rope_out"] = self.b["d_q_rope"] if in_place else P.upload(np.full((T, self.os), 5.0), x)
        if status:
            self.b["d_status"] = hip.DeviceBuffer.from_array(np.zeros(1, np.uint32))
        c = paged.Cache(d_rows=self.cache.ptr, dtype=paged.TYPE[cache], n_pages=n_pages, page_size=ps, kv_lora_rank=L,
                        qk_rope=RP, row_stride=self.stride)
        self.args = paged.RowWrite(cache=c, dtype=paged.TYPE[x], n_tokens=T, n_heads=H, eps=self.eps, rope_theta=self.theta,
                                   kv_stride=self.ks, q_stride=self.qs, q_out_stride=self.os, n_kv=n_kv,
                                   **{k: v.ptr for k, v in self.b.items()})

    def status(self):
        return int(self.b["d_status"].download(np.uint32)[0])

    def check(self, passed=()):
        """Every row and query but the tokens `passed` over. A norm of L squares in f32 is off by (L / 2 + 8) u, a
        turned value by 8 u of its pair's length (cos and sin to 2 u each, two products, a sum)."""
        u_c, u_x = (P.U16 if t == "bf16" else P.U32 for t in (self.ct, self.x))
        rows, want, far = P.download(self.cache, self.ct, self.rows0.shape), self.rows0.astype(np.float64), \
            np.zeros(self.rows0.shape)
        for t in range(self.T):
            if t in passed or self.slot[t] < 0:
                continue
            kv = self.kv[t if self.src is None else self.src[t], :self.W]
            row = P.latent_row(kv, self.w, self.eps, self.L, int(self.pos[t]), self.theta)
            half, n = self.RP // 2, np.hypot(kv[self.L::2].astype(np.float64), kv[self.L + 1::2])
            size = np.concatenate([np.abs(row[:self.L]) * (self.L / 2 + 8), 8 * n, 8 * n])
            want[self.slot[t], :self.W] = row
            far[self.slot[t], :self.W] = size * P.U32 * 1.01 + u_c * np.abs(row) * (1 + 1e-3)
            assert len(n) == half
        assert np.all(np.abs(rows - want) <= far)
        if self.H:
            out = P.download(self.b["d_q_rope_out"], self.x, (self.T, self.os))
            q = self.q[:, :self.H * self.RP].reshape(self.T, self.H, self.RP)
            want = P.rope(q, self.pos[:, None], self.theta)
            n = np.hypot(q[..., 0::2].astype(np.float64), q[..., 1::2])
            far = 8.1 * P.U32 * np.concatenate([n, n], -1) + u_x * np.abs(want) * (1 + 1e-3)
            ok = np.abs(out[:, :self.H * self.RP].reshape(want.shape) - want) <= far
            skip = [t for t in passed if self.pos[t] < 0]
            ok[skip] = True
            assert ok.all()
            if self.os > self.H * self.RP and self.b["d_q_rope_out"] is not self.b["d_q_rope"]:
                assert np.all(out[:, self.H * self.RP:] == 5.0)


@pytest.mark.parametrize("x,cache", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("T,L,RP,H,ps,pad", [(1, 512, 64, 64, 64, 0), (1, 8, 8, 0, 8, 8), (7, 96, 24, 5, 16, 16),
                                             (333, 256, 32, 20, 32, 8), (1030, 504, 56, 3, 8, 0)])
def test_write(gpu, T, L, RP, H, ps, pad, x, cache):
    w = Write(T + L, T, x, cache, L, RP, H, ps, pad)
    paged.write_rows(w.args)
    hip.synchronize()
    w.check()
    assert w.status() == 0


@pytest.mark.parametrize("x,cache", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("T,RP,H", [(5, 64, 1), (5, 64, 9), (5, 64, 20), (1100, 64, 64), (3, 40, 1024)])
def test_write_waves_of_a_token(gpu, T, RP, H, x, cache):
    """One to four waves share a token's heads."""
    w = Write(H, T, x, cache, 128, RP, H, 16, 8)
    paged.write_rows(w.args)
    hip.synchronize()
    w.check()
    assert w.status() == 0


def test_write_far_positions(gpu):
    w = Write(1, 6, "f32", "f32", 64, 64, 2, 16, pos=[0, 1, 131071, 1 << 20, (1 << 30) + 12345, 2 ** 31 - 1])
    paged.write_rows(w.args)
    hip.synchronize()
    w.check()


@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_write_queries_in_place(gpu, x):
    w = Write(2, 50, x, "bf16", 128, 40, 17, 16, in_place=True, status=False)
    paged.write_rows(w.args)
    hip.synchronize()
    w.check()


def test_write_accepted_rows_again(gpu):
    """The rows of accepted nodes from the same projections at other slots; one slot is none."""
    w = Write(3, 4, "f32", "bf16", 64, 16, 0, 16, src=[9, 0, 0, 5], n_kv=10, slot=[3, 17, -1, 0])
    paged.write_rows(w.args)
    hip.synchronize()
    w.check()
    assert w.status() == 0


@pytest.mark.parametrize("x,cache", [("f32", "f32"), ("bf16", "bf16")])
def test_write_sources_behind_the_tokens(gpu, x, cache):
    """A step captured with room for more writes rows again: what stands in d_src where the slots are -1 is not looked
    at, and no flaw."""
    w = Write(39, 7, x, cache, 64, 16, 2, 16, src=[2, 0, 3, -1, 4, 2 ** 31 - 1, -7], n_kv=4, slot=[5, 9, 0, -1, -1, -1, -1])
    paged.write_rows(w.args)
    hip.synchronize()
    w.check()
    assert w.status() == 0


def test_write_flaws(gpu):
    w = Write(4, 6, "f32", "f32", 64, 16, 3, 16, n_pages=2, src=[0, 1, -1, 7, 3, 4], n_kv=7,
              slot=[32, -2, 4, 5, 6, 7], pos=[4, 5, 6, 7, -1, 8])
    paged.write_rows(w.args)
    hip.synchronize()
    w.check(passed=(0, 1, 2, 3, 4))
    assert w.status() == paged.E_SLOT | paged.E_LEN


# ---- attention -----------------------------------------------------------------
class Tree:
    """Requests over one cache. lens, adds: as wl_paged_map's; masks: None (chains) or 64-bit ints per token."""

    def __init__(self, seed, q, cache, L, RP, H, ps, lens, adds, masks=None, pad=0, tail=0, spread=2.0, row_pad=0,
                 first_page=0, page_order=None, fill=np.nan):
        rng = np.random.default_rng(seed)
        W, R = L + RP, len(lens)
        self.qt, self.ct, self.L, self.W, self.H, self.ps, self.lens, self.adds = q, cache, L, W, H, ps, lens, adds
        held = [-(-(n + a) // ps) for n, a in zip(lens, adds)]
        self.max_pages, self.n_pages = max(held + [1]), first_page + sum(held) + 1
        order = rng.permutation(sum(held) + 1) + first_page
        self.table = np.full((R, self.max_pages), -1, np.int32)  # entries behind a request's pages are never looked at
        self.rows = []
        self.stride = W + row_pad
        small = self.n_pages - first_page
        pages = np.full((small, ps, self.stride), fill, np.float32)  # rows that belong to nobody
        at = 0
        for r in range(R):
            self.table[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
            n = lens[r] + adds[r]
            rows = P.as_type(rng.standard_normal((n, W)), cache)
            self.rows.append(rows)
            for k in range(n):
                pages[self.table[r, k // ps] - first_page, k % ps, :W] = rows[k]
        self.scale = 1.0 / np.sqrt(192.0 + RP)
        self.T = sum(adds) + tail
        sd = spread / (self.scale * np.sqrt(W))
        self.ql = P.as_type(sd * rng.standard_normal((self.T, H * L + pad)), q)
        self.qr = P.as_type(sd * rng.standard_normal((self.T, H * RP + 2 * pad)), q)
        self.os = H * L + 3 * pad
        self.cu = np.concatenate([[0], np.cumsum(adds)]).astype(np.int32)
        self.masks = masks
        self.pages, self.first_page = pages, first_page

    def upload(self, **change):
        es = 2 if self.ct == "bf16" else 4
        page_bytes = self.ps * self.stride * es
        self.cache = hip.DeviceBuffer(self.n_pages * page_bytes)
        self.cache.upload(P.bf16_bits(self.pages) if self.ct == "bf16" else self.pages, self.first_page * page_bytes)
        i32 = lambda x: hip.DeviceBuffer.from_array(np.asarray(x, np.int32).reshape(-1))  # noqa: E731
        self.b = dict(d_q_lat=P.upload(self.ql, self.qt), d_q_rope=P.upload(self.qr, self.qt),
                      d_out=P.upload(np.full((self.T, self.os), 7.0), self.qt), d_table=i32(change.get("table", self.table)),
                      d_len=i32(change.get("lens", self.lens)), d_cu=i32(change.get("cu", self.cu)), d_status=i32([0]))
        if self.masks is not None:
            self.b["d_mask"] = hip.DeviceBuffer.from_array(np.array(self.masks + [0] * (self.T - len(self.masks)), np.uint64))
        c = paged.Cache(d_rows=self.cache.ptr, dtype=paged.TYPE[self.ct], n_pages=self.n_pages, page_size=self.ps,
                        kv_lora_rank=self.L, qk_rope=self.W - self.L, row_stride=self.stride)
        self.args = paged.TreeAttention(cache=c, dtype=paged.TYPE[self.qt], n_req=len(self.lens), n_tokens=self.T,
                                        n_heads=self.H, max_pages=self.max_pages, scale=self.scale,
                                        q_lat_stride=self.ql.shape[1], q_rope_stride=self.qr.shape[1],
                                        out_stride=self.os, **{k: v.ptr for k, v in self.b.items()})
        n = paged.tree_attention_scratch(self.args)
        self.b["d_scratch"] = hip.DeviceBuffer(n)
        self.b["d_scratch"].upload(np.full(n, 0xFF, np.uint8))  # NaN wherever it is not written first
        self.args.d_scratch, self.args.scratch_bytes = self.b["d_scratch"].ptr, n
        return self

    def run(self, stream=0):
        paged.tree_attention(self.args, stream)
        hip.synchronize()
        return self

    def status(self):
        return int(self.b["d_status"].download(np.uint32)[0])

    def out(self):
        return P.download(self.b["d_out"], self.qt, (self.T, self.os))

    def want(self, r, i):
        """(output, bound) of node i of request r, [H, L] each."""
        t, n, a = self.cu[r] + i, self.lens[r], self.adds[r]
        bits = (2 << i) - 1 if self.masks is None else int(self.masks[t])
        seen = np.array([True] * n + [bool(bits >> j & 1) for j in range(a)], bool)
        q = np.concatenate([self.ql[t, :self.H * self.L].reshape(self.H, self.L),
                            self.qr[t, :self.H * (self.W - self.L)].reshape(self.H, -1)], 1)
        return P.tree_attention(q, self.rows[r], self.L, self.scale, seen, self.qt)

    def check(self, skip=(), nan=()):
        """Every request's rows but those of `skip` (left as they were) and `nan` (all NaN), and what nobody writes."""
        out = self.out()
        assert np.all(out[self.cu[-1]:] == 7.0) and np.all(out[:, self.H * self.L:] == 7.0)
        for r, a in enumerate(self.adds):
            for i in range(a):
                got = out[self.cu[r] + i, :self.H * self.L].reshape(self.H, self.L)
                if r in skip:
                    assert np.all(got == 7.0)
                elif r in nan:
                    assert np.isnan(got).all()
                else:
                    y, far = self.want(r, i)
                    assert np.all(np.abs(got - y) <= far), (r, i, np.max(np.abs(got - y) / far))


class Mean(Tree):
    """A Tree whose bound is that of a mean by rounded weights."""
    def want(self, r, i):
        t, n, a = self.cu[r] + i, self.lens[r], self.adds[r]
        bits = (2 << i) - 1 if self.masks is None else int(self.masks[t])
        seen = np.array([True] * n + [bool(bits >> j & 1) for j in range(a)], bool)
        q = np.concatenate([self.ql[t, :self.H * self.L].reshape(self.H, self.L),
                            self.qr[t, :self.H * (self.W - self.L)].reshape(self.H, -1)], 1)
        return P.tree_attention_mean(q, self.rows[r], self.L, self.scale, seen, self.qt)


def random_trees(rng, adds):
    masks = []
    for a in adds:
        m = []
        for i in range(a):
            p = int(rng.integers(-1, i)) if i else -1
            m.append((1 << i) | (m[p] if p >= 0 else 0))
        masks += m
    return masks


TYPES = [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")]
SHAPES = [(512, 64, 64, 64), (512, 64, 16, 16), (256, 32, 20, 32), (128, 64, 128, 64), (96, 8, 1, 8), (200, 40, 7, 8),
          (512, 64, 33, 1024), (8, 8, 3, 8)]


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("L,RP,H,ps", SHAPES)
def test_attention(gpu, L, RP, H, ps, q, cache):
    rng = np.random.default_rng(L + H)
    lens = [0, 1, 63, 130, 0, 517]
    adds = [1, 3, 0, 13, 5, 2]
    Tree(L + RP + H, q, cache, L, RP, H, ps, lens, adds, random_trees(rng, adds), tail=2).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_chains_strides(gpu, q, cache):
    lens, adds = [40, 3, 300, 64], [64, 1, 9, 32]
    t = Tree(5, q, cache, 512, 64, 8, 16, lens, adds, pad=24, row_pad=40, tail=1).upload().run()
    t.check()
    assert t.status() == 0


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 1023])
def test_attention_one_token(gpu, q, cache, n):
    """The form for decoding: one request, one token, lengths around every tile's edge (n keys with its own)."""
    Tree(n, q, cache, 512, 64, 64, 64, [n - 1], [1]).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_long_and_uneven(gpu, q, cache):
    """Splits that end inside requests: a long context among short ones, a full tree."""
    rng = np.random.default_rng(8)
    lens, adds = [20011, 5, 700, 0, 9000], [1, 2, 64, 1, 3]
    Tree(9, q, cache, 512, 64, 4, 64, lens, adds, random_trees(rng, adds)).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("H,lens,adds", [(20, [900, 0, 333, 4000], [5, 1, 64, 9]), (64, [2500], [7]), (33, [31, 0, 64], [2, 0, 3]),
                                         (64, list(range(0, 1200, 20)), [2] * 60), (128, [70, 2100], [64, 1])],
                         ids=["uneven", "one", "short", "sixty", "tall"])
def test_attention_pieces(gpu, q, cache, H, lens, adds):
    """Fewer row tiles than work-groups: each has a piece of one."""
    rng = np.random.default_rng(21)
    Tree(22, q, cache, 128, 32, H, 16, lens, adds, random_trees(rng, adds)).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("H,lens,adds,R", [(64, [2500], [7], 64), (20, [900, 333, 4000], [5, 64, 9], 64), (128, [70, 2100], [64, 1], 250)])
def test_attention_requests_without_tokens_change_nothing(gpu, q, cache, H, lens, adds, R):
    """A step with room for R requests of which a few are live: the others' results, bit for bit, of a call of the live
    ones alone."""
    a = Mean(35, q, cache, 128, 32, H, 16, lens, adds)
    alone = a.upload().run().out()
    at = [(k + 1) * R // (len(lens) + 1) for k in range(len(lens))]  # the live ones' places
    b = Mean(35, q, cache, 128, 32, H, 16, [lens[at.index(r)] if r in at else 0 for r in range(R)],
             [adds[at.index(r)] if r in at else 0 for r in range(R)])
    assert np.array_equal(a.ql, b.ql) and np.array_equal(a.pages, b.pages, equal_nan=True)
    assert np.array_equal(b.upload().run().out(), alone)
    b.check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_refused_among_pieces(gpu, q, cache):
    lens, adds = [2000, 300, 9, 1400], [2, 3, 1, 2]
    def tree():
        return Tree(23, q, cache, 128, 16, 70, 16, lens, adds, tail=3)
    t = tree()
    table = t.table.copy()
    table[0, 77] = -3
    t.upload(table=table).run().check(nan=(0,))
    assert t.status() == paged.E_PAGE
    t = tree()
    t.upload(lens=[2000, -5, 9, 2 ** 31 - 1]).run().check(nan=(1, 3))
    assert t.status() == paged.E_LEN
    t = tree()
    t.upload(cu=[0, 2, 5, 6, 12]).run().check(skip=(3,))
    assert t.status() == paged.E_LEN


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_many_requests(gpu, q, cache):
    rng = np.random.default_rng(10)
    R = 300
    lens, adds = [int(x) for x in rng.integers(0, 50, R)], [int(x) for x in rng.integers(0, 3, R)]
    Tree(11, q, cache, 128, 16, 4, 16, lens, adds, random_trees(rng, adds)).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("R", [600, 1500, 4096])
def test_attention_requests_beyond_a_thread_each(gpu, q, cache, R):
    rng = np.random.default_rng(R)
    lens, adds = [int(x) for x in rng.integers(0, 40, R)], [int(x) for x in rng.integers(0, 3, R)]
    Tree(24, q, cache, 64, 8, 2, 8, lens, adds, random_trees(rng, adds)).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("scale", [-0.07, 0.0])
def test_attention_scales_that_are_not_positive(gpu, q, cache, scale):
    rng = np.random.default_rng(25)
    lens, adds = [70, 0, 611], [5, 2, 33]
    t = Tree(26, q, cache, 96, 16, 5, 16, lens, adds, random_trees(rng, adds))
    t.scale = scale
    t.upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_magnitudes(gpu, q, cache):
    """Large queries against small rows, scaled by powers of two: exact in every type."""
    t = Tree(27, q, cache, 128, 32, 6, 16, [300, 40], [3, 9])
    t.ql, t.qr = t.ql * np.float32(2.0 ** 60), t.qr * np.float32(2.0 ** 60)
    t.rows = [x * np.float32(2.0 ** -60) for x in t.rows]
    t.pages = t.pages * np.float32(2.0 ** -60)
    t.upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("H,n", [(4, 500), (64, 1500)])
def test_attention_large_rows_with_rising_scores(gpu, q, cache, H, n):
    """Rows of some 2^66 against queries of 2^-66 (exact scalings): scores that rise by some 50 powers of two from a
    tile of keys to the next, so that weights relative to an early tile, times the values, are beyond f32 where the
    result is not."""
    for sign in (1.0, -1.0):
        t = Mean(32, q, cache, 128, 16, H, 16, [n], [2])
        ramp = P.as_type(sign * 30.0 * (np.arange(n + 2) % 500 - 250) / 250, "bf16")
        for k in range(n + 2):
            t.rows[0][k, 128] = ramp[k]
            t.pages[t.table[0, k // 16], k % 16, 128] = ramp[k]
        t.qr[:, 0::16] = 128.0
        t.ql, t.qr = t.ql * np.float32(2.0 ** -66), t.qr * np.float32(2.0 ** -66)
        t.rows = [x * np.float32(2.0 ** 66) for x in t.rows]
        t.pages = t.pages * np.float32(2.0 ** 66)
        t.upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("L,H,lens,adds", [(128, 4, [40, 900], [1, 3]), (512, 64, [5000], [1]), (256, 20, [700] * 40, [2] * 40),
                                           (96, 16, [90] * 300, [1] * 300)], ids=["short", "parts", "pieces", "whole"])
def test_attention_values_at_the_end_of_the_range(gpu, q, cache, L, H, lens, adds):
    """Latent values next to the largest bf16 number, scores of the rotary parts alone: any result lies between the
    values, whatever their unnormalised sums come to. (A call that is off by more than half a bf16 step of the largest
    would give an infinity, which no bound lets pass.)"""
    top = float(np.float32(2.0 ** 127 * (2 - 2.0 ** -7)))
    for signs in (1.0, -1.0), (1.0, 1.0):
        t = Mean(33, q, cache, L, 16, H, 16, lens, adds)
        rng = np.random.default_rng(34)
        t.ql[:] = 0.0
        for r, rows in enumerate(t.rows):
            n = len(rows)
            big = np.where(rng.random((n, 1)) < 0.5, signs[0], signs[1]) * top * (1 - 0.1 * rng.random((n, L)))
            rows[:, :L] = np.clip(P.as_type(big, cache), -top, top)
            rows[:n // 2, :L] = np.where(rng.random((n // 2, 1)) < 0.5, signs[0], signs[1]) * top
            for k in range(n):
                t.pages[t.table[r, k // 16], k % 16, :L] = rows[k, :L]
        t.upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_most_heads(gpu, q, cache):
    rng = np.random.default_rng(28)
    Tree(29, q, cache, 16, 8, 1024, 8, [40, 3], [2, 1], random_trees(rng, [2, 1])).upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_rows_that_see_nothing(gpu, q, cache):
    """Masks of nothing: zeros without a context, the context alone with one. Any 64-bit mask, not only a tree's."""
    rng = np.random.default_rng(12)
    lens, adds = [0, 70, 0, 3], [4, 4, 64, 64]
    masks = [0, 2, 0, 15] + [0, 8, 1, 0] + [int(x) for x in rng.integers(0, 1 << 62, 64)] + [0, (1 << 64) - 1] + \
        [1 << int(x) for x in rng.integers(0, 64, 62)]
    t = Tree(13, q, cache, 256, 64, 6, 16, lens, adds, masks).upload().run()
    t.check()
    assert np.all(t.out()[0, :6 * 256] == 0.0)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_attention_flawed_rows_reach_those_that_see_them(gpu, q, cache, value):
    """Node 1's row holds a NaN or an infinity: its descendants are not finite, everyone else exact."""
    masks = [1, 3, 5, 11, 21, 1 << 5]
    for n in (0, 61, 200):
        t = Tree(14 + n, q, cache, 512, 64, 5, 32, [n, n], [6, 6], masks + masks)
        k = n + 1
        t.pages[t.table[0, k // 32], k % 32, 100] = value
        t.upload().run()
        out = t.out()[:, :5 * 512].reshape(12, 5, 512)
        for i in range(12):
            if i in (1, 3):
                assert not np.isfinite(out[i]).all(axis=1).any()
            else:
                y, far = t.want(i // 6, i % 6)
                assert np.all(np.abs(out[i] - y) <= far)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("spread", [0.0, 60.0, 2000.0])
def test_attention_far_apart_scores(gpu, q, cache, spread):
    """From equal scores to weights that are all but one zero; the largest score late and early."""
    lens, adds = [700, 133], [2, 5]
    t = Tree(15, q, cache, 512, 64, 3, 64, lens, adds, spread=spread)
    if spread > 1000:  # the bound covers 32-bit scores' own errors, which weights of this spread magnify
        t.upload().run()
        assert np.isfinite(t.out()).all() and t.status() == 0
        return
    t.upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_rising_scores(gpu, q, cache):
    """Scores that rise (or fall) by hundreds along the keys: the running maximum moves in every tile."""
    for sign in (1.0, -1.0):
        t = Tree(16, q, cache, 128, 16, 4, 16, [500], [2])
        n = 502
        ramp = P.as_type(sign * np.linspace(-30, 30, n), "bf16")
        for k in range(n):
            t.rows[0][k, 128] = ramp[k]
            t.pages[t.table[0, k // 16], k % 16, 128] = ramp[k]
        t.qr[:, 0::16] = 128.0
        t.upload().run().check()


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("lens,adds", [([9000], [2]), ([9000] + [1000] * 300, [2] + [1] * 300)], ids=["parts", "whole"])
def test_attention_scores_that_rise_by_more_than_a_walk_can_hold(gpu, q, cache, lens, adds):
    """Scores that rise by 70 powers of two from a tile of 32 keys to the next, in ramps of 11 tiles: every longer walk
    is done again, the ones of five tiles and more around the ring of four, and every ramp's top counts."""
    t = Mean(36, q, cache, 128, 16, 64 if len(lens) > 1 else 256, 16, lens, adds, spread=0.5)
    n = max(lens) + max(adds)
    powers = 70.0 * (np.arange(n) % (11 * 32)) / 32
    t.qr[:, 0::16] = 128.0
    ramp = P.as_type((powers - 385) * np.log(2) / (128 * t.scale), "bf16")
    assert np.ptp(ramp[:32].astype(np.float64)) * 128 * t.scale / np.log(2) > 66
    for r, rows in enumerate(t.rows):
        rows[:, 128] = ramp[:len(rows)]
        for k in range(len(rows)):
            t.pages[t.table[r, k // 16], k % 16, 128] = ramp[k]
    t.upload().run().check()


@pytest.mark.parametrize("L,RP,H,lens,adds", [(256, 64, 4, [30, 0, 500], [3, 1, 2]), (200, 40, 4, [9000], [3]), (136, 8, 1, [700] * 280, [1] * 280),
                                              (256, 64, 8, [40000, 5, 6], [1, 2, 1])], ids=["short", "parts", "whole", "long"])
def test_attention_few_rows_and_a_middling_latent_part(gpu, L, RP, H, lens, adds):
    """16-bit calls of at most 32 rows a request with latent parts of 129 to 256 columns, whole row tiles and parts."""
    rng = np.random.default_rng(37)
    Mean(38, "bf16", "bf16", L, RP, H, 16, lens, adds, random_trees(rng, adds)).upload().run().check()


def test_attention_refused_requests(gpu):
    """Flaws that only the device sees spoil their own request and set their bit; everyone else is exact."""
    lens, adds = [20, 30, 9, 40], [2, 3, 1, 2]
    for q, cache in TYPES:
        def tree():
            return Tree(17, q, cache, 128, 16, 6, 16, lens, adds, tail=3)
        t = tree()
        table = t.table.copy()
        table[1, 1] = t.n_pages
        t.upload(table=table).run().check(nan=(1,))
        assert t.status() == paged.E_PAGE
        t = tree()
        table[1, 1], table[3, 0] = t.table[1, 1], -1
        t.upload(table=table).run().check(nan=(3,))
        assert t.status() == paged.E_PAGE
        t = tree()
        t.upload(lens=[20, -5, 9, 2 ** 31 - 1]).run().check(nan=(1, 3))
        assert t.status() == paged.E_LEN
        t = tree()
        t.upload(lens=[20, 30, t.max_pages * 16, 40]).run().check(nan=(2,))  # one key more than the row has entries for
        assert t.status() == paged.E_LEN
        t = tree()
        t.upload(cu=[0, 2, 5, 6, 12]).run().check(skip=(3,))  # the last range ends behind the arrays
        assert t.status() == paged.E_LEN


def test_attention_too_many_nodes(gpu):
    for q, cache in TYPES:
        t = Tree(18, q, cache, 128, 16, 3, 16, [4, 8], [65, 2], [1] * 67).upload().run()
        t.check(nan=(0,))
        assert t.status() == paged.E_TREE


@pytest.mark.parametrize("q,cache", TYPES)
def test_attention_offsets_past_32_bits(gpu, q, cache):
    """Pages behind the first 4 GiB of a cache: byte and element offsets pass 32 bits."""
    first = (1 << 33) // (64 * 576 * (2 if cache == "bf16" else 4)) + 1
    t = Tree(19, q, cache, 512, 64, 2, 64, [150], [3], first_page=first)
    t.upload().run().check()
    t.cache.free()


def test_calls_on_streams_and_in_graphs(gpu):
    """A step's three calls on a stream of their own, beside the same calls on another; then captured, each graph with
    its own scratch, and replayed among eager calls: the same bits every time."""
    def step(seed, q, cache):
        rng = np.random.default_rng(seed)
        lens, adds = [900, 5, 64], [9, 1, 17]
        return Tree(seed, q, cache, 512, 64, 16, 64, lens, adds, random_trees(rng, adds)).upload()
    a, b = step(20, "bf16", "bf16"), step(21, "f32", "f32")
    s1, s2 = hip.Stream(), hip.Stream()
    for _ in range(5):
        paged.tree_attention(a.args, s1.handle)
        paged.tree_attention(b.args, s2.handle)
    hip.synchronize()
    a.check()
    b.check()
    first = a.out(), b.out()
    graphs = []
    for t, s in ((a, s1), (b, s2)):
        g = hip.Graph(s)
        g.begin()
        paged.tree_attention(t.args, s.handle)
        g.end()
        graphs.append(g)
    m_step = make_step(np.random.default_rng(5), 37, 16, 64, 300, True)
    m = P.Map(**m_step)
    w = Write(6, 300, "f32", "bf16", 256, 32, 20, 32)
    g = hip.Graph(s1)
    g.begin()
    paged.page_map(m.args, s1.handle)
    paged.write_rows(w.args, s1.handle)
    g.end()
    graphs.append(g)
    for k in range(4):
        for t in (a, b):
            t.b["d_out"].upload(np.zeros(t.b["d_out"].nbytes, np.uint8))
        for g in graphs:
            g.launch()
        hip.synchronize()
        assert np.array_equal(a.out(), first[0]) and np.array_equal(b.out(), first[1])
        check_step(m, m_step)
        w.check()
        paged.tree_attention(a.args)  # eager work between the replays
        hip.synchronize()
        assert np.array_equal(a.out(), first[0])
    for g in graphs:
        g.destroy()
    s1.destroy()
    s2.destroy()


# ---- together ------------------------------------------------------------------
@pytest.mark.parametrize("x,cache", [("f32", "f32"), ("bf16", "bf16")])
def test_steps_of_a_serving_loop(gpu, x, cache):
    """Prompts are taken up, trees drafted, verified and partly accepted, requests end and others take their pages: map,
    write and attention of every step against the requests' token histories."""
    rng = np.random.default_rng(30)
    L, RP, H, ps, R, max_pages, n_pages, theta, eps = 128, 32, 6, 16, 4, 12, 30, 1e4, 1e-6
    W = L + RP
    norm = P.as_type(1 + 0.1 * rng.standard_normal(L), "bf16")
    d_norm, d_cache = P.upload(norm, "bf16"), P.upload(np.full((n_pages * ps, W), np.nan), cache)
    c = paged.Cache(d_rows=d_cache.ptr, dtype=paged.TYPE[cache], n_pages=n_pages, page_size=ps, kv_lora_rank=L, qk_rope=RP,
                    row_stride=W)
    table, free, n_free = np.full((R, max_pages), -1, np.int32), np.arange(n_pages, dtype=np.int32), n_pages
    have, hist = [0] * R, [[] for _ in range(R)]  # a request's accepted rows, as the cache holds them
    scale = 0.1

    def run(lens, adds, parent, kv, src=None, attend=True):
        """One map and write (and attention) of the step; (slots, positions, masks, outputs)."""
        nonlocal table, free, n_free, have
        m = P.Map(ps, n_pages, max_pages, lens, adds, have, free, n_free, table, parent)
        paged.page_map(m.args)
        T = sum(adds)
        ql, qr = (P.as_type(3 * rng.standard_normal((T, H * n)), x) for n in (L, RP))
        b = dict(d_kv=P.upload(kv, x), d_q_rope=P.upload(qr, x), d_q_rope_out=P.upload(np.zeros_like(qr), x),
                 d_q_lat=P.upload(ql, x), d_out=P.upload(np.zeros_like(ql), x))
        if src is not None:
            b["d_src"] = hip.DeviceBuffer.from_array(np.asarray(src, np.int32))
        w = paged.RowWrite(cache=c, dtype=paged.TYPE[x], n_tokens=T, n_heads=H, eps=eps, rope_theta=theta, kv_stride=W,
                           d_kv=b["d_kv"].ptr, d_norm_w=d_norm.ptr, d_pos=m.b["d_pos"].ptr, d_slot=m.b["d_slot"].ptr,
                           d_src=b["d_src"].ptr if src is not None else None, n_kv=len(kv), d_q_rope=b["d_q_rope"].ptr,
                           q_stride=H * RP, d_q_rope_out=b["d_q_rope_out"].ptr, q_out_stride=H * RP,
                           d_status=m.b["d_status"].ptr)
        paged.write_rows(w)
        out = None
        if attend:
            a = paged.TreeAttention(cache=c, dtype=paged.TYPE[x], n_req=R, n_tokens=T, n_heads=H, max_pages=max_pages,
                                    scale=scale, d_q_lat=b["d_q_lat"].ptr, q_lat_stride=H * L,
                                    d_q_rope=b["d_q_rope_out"].ptr, q_rope_stride=H * RP, d_out=b["d_out"].ptr,
                                    out_stride=H * L, d_table=m.b["d_table"].ptr, d_len=m.b["d_len"].ptr,
                                    d_cu=m.b["d_cu"].ptr, d_mask=m.b["d_mask"].ptr if "d_mask" in m.b else None,
                                    d_status=m.b["d_status"].ptr)
            n = paged.tree_attention_scratch(a)
            b["d_scratch"] = hip.DeviceBuffer(n)
            a.d_scratch, a.scratch_bytes = b["d_scratch"].ptr, n
            paged.tree_attention(a)
            out = P.download(b["d_out"], x, (T, H, L))
        hip.synchronize()
        assert m.get("status")[0] == 0
        table, free, n_free, have = m.get("table"), m.get("free"), int(m.get("n_free_out")[0]), m.get("have_out").tolist()
        owned = [int(p) for r in range(R) for p in table[r, :have[r]]] + free[:n_free].tolist()
        assert sorted(owned) == list(range(n_pages))  # every page has one holder
        q = np.concatenate([ql.reshape(T, H, L), P.download(b["d_q_rope_out"], x, (T, H, RP))], -1)
        return m.get("slot"), m.get("pos"), m.get("mask") if parent is not None else None, q, out

    for step in range(6):
        lens = [len(h) for h in hist]
        adds = [int(v) for v in rng.integers(1, 12, R)]
        if step == 3:  # request 2 ends; its pages go back
            hist[2], lens[2], adds[2] = [], 0, 0
        parent = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(a)] for a in adds] + [[]]).astype(np.int32)
        kv = P.as_type(rng.standard_normal((sum(adds), W)), x)
        slot, pos, mask, q, out = run(lens, adds, parent, kv)
        rows = P.download(d_cache, cache, (n_pages * ps, W))[slot]  # as the cache holds them
        u = P.U16 if cache == "bf16" else P.U32
        exact = P.latent_row(kv, norm, eps, L, pos, theta)
        assert np.all(np.abs(rows - exact) <= u * np.abs(exact) * 1.01 + (L / 2 + 16) * P.U32 * (np.abs(exact) + 4))
        t, accepted = 0, []
        for r, a in enumerate(adds):
            keys = np.array(hist[r] + list(rows[t:t + a])).reshape(-1, W)
            for i in range(a):
                bits = int(mask[t + i])
                seen = np.array([True] * lens[r] + [bool(bits >> j & 1) for j in range(a)], bool)
                y, far = P.tree_attention(q[t + i], keys, L, scale, seen, x)
                assert np.all(np.abs(out[t + i] - y) <= far)
            # a random node's path is accepted
            tip = int(mask[t + int(rng.integers(0, a))]) if a else 0
            path = [j for j in range(a) if tip >> j & 1]
            accepted.append([t + j for j in path])
            t += a
        # the accepted nodes' rows move up behind the context: the same projections, their final slots
        src = [j for path in accepted for j in path]
        n_acc = [len(path) for path in accepted]
        if src:
            slot2, pos2, _, _, _ = run(lens, n_acc, None, kv, src=src, attend=False)
            assert np.array_equal(pos2, pos[src])
            again = P.download(d_cache, cache, (n_pages * ps, W))[slot2]
            assert np.array_equal(again, rows[src])  # bit for bit
            t = 0
            for r, n in enumerate(n_acc):
                hist[r] += list(again[t:t + n])
                t += n
