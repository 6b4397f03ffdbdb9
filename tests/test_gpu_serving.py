"""Steps of a serving loop over a 4-bit cache, through a window, with the drafted tokens' log probabilities; and the
calls on streams and in graphs."""
import numpy as np
import pytest

from windlass_amd import hip, paged

from . import paged_ref as P
from . import serving_ref as S
from .test_gpu_mx4 import Write, i32
from .test_gpu_paged import random_trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (17, 3)])
def test_steps_of_a_serving_loop(gpu, x, window, sinks):
    """Prompts are taken up, trees drafted, scored and accepted where they are likely: every call of every step against
    the requests' histories, and each request's rows read back at the end."""
    rng = np.random.default_rng(30)
    L, RP, H, ps, R, V, max_pages, n_pages, theta, eps, scale = 128, 32, 6, 16, 4, 3001, 12, 40, 1e4, 2.0 ** -20, 0.1
    W, stride = L + RP, S.row_bytes(128, 32)
    norm = P.as_type(1 + 0.1 * rng.standard_normal(L), "bf16")
    head = rng.standard_normal((H * L, V)) / 8
    d_norm = P.upload(norm, "bf16")
    d_cache = hip.DeviceBuffer.from_array(np.full((n_pages * ps, stride), 0xFF, np.uint8))
    c = paged.Cache(d_rows=d_cache.ptr, dtype=paged.TYPE["mxfp4"], n_pages=n_pages, page_size=ps, kv_lora_rank=L, qk_rope=RP,
                    row_stride=stride)
    table, free, n_free = np.full((R, max_pages), -1, np.int32), np.arange(n_pages, dtype=np.int32), n_pages
    have, hist = [0] * R, [[] for _ in range(R)]  # a request's accepted rows, as values

    def cached(slots):
        code, e, rope = S.unpack(d_cache.download(np.uint8).reshape(-1, stride)[slots], L)
        return np.concatenate([S.values(code, e), rope], 1)

    def step(lens, adds, parent, kv, src=None):
        nonlocal table, free, n_free, have
        m = P.Map(ps, n_pages, max_pages, lens, adds, have, free, n_free, table, parent)
        paged.page_map(m.args)
        T = sum(adds)
        ql, qr = (P.as_type(3 * rng.standard_normal((T, H * n)), x) for n in (L, RP))
        b = dict(d_kv=P.upload(kv, x), d_q_rope=P.upload(qr, x), d_q_rope_out=P.upload(np.zeros_like(qr), x),
                 d_q_lat=P.upload(ql, x), d_out=P.upload(np.zeros_like(ql), x))
        if src is not None:
            b["d_src"] = i32(src)
        paged.write_rows(paged.RowWrite(
            cache=c, dtype=paged.TYPE[x], n_tokens=T, n_heads=H, eps=eps, rope_theta=theta, kv_stride=W, d_kv=b["d_kv"].ptr,
            d_norm_w=d_norm.ptr, d_pos=m.b["d_pos"].ptr, d_slot=m.b["d_slot"].ptr, n_kv=len(kv),
            d_src=b["d_src"].ptr if src is not None else None, d_q_rope=b["d_q_rope"].ptr, q_stride=H * RP,
            d_q_rope_out=b["d_q_rope_out"].ptr, q_out_stride=H * RP, d_status=m.b["d_status"].ptr))
        out = None
        if src is None:
            a = paged.TreeAttention(cache=c, dtype=paged.TYPE[x], n_req=R, n_tokens=T, n_heads=H, max_pages=max_pages,
                                    scale=scale, d_q_lat=b["d_q_lat"].ptr, q_lat_stride=H * L, d_q_rope=b["d_q_rope_out"].ptr,
                                    q_rope_stride=H * RP, d_out=b["d_out"].ptr, out_stride=H * L, d_table=m.b["d_table"].ptr,
                                    d_len=m.b["d_len"].ptr, d_cu=m.b["d_cu"].ptr, d_mask=m.b["d_mask"].ptr,
                                    d_status=m.b["d_status"].ptr)
            n = paged.tree_attention_scratch(a)
            b["d_scratch"] = hip.DeviceBuffer(n)
            a.d_scratch, a.scratch_bytes = b["d_scratch"].ptr, n
            paged.window_attention(paged.WindowAttention(tree=a, window=window, n_sinks=sinks))
            out = P.download(b["d_out"], x, (T, H, L))
        hip.synchronize()
        assert m.get("status")[0] == 0
        table, free, n_free, have = m.get("table"), m.get("free"), int(m.get("n_free_out")[0]), m.get("have_out").tolist()
        q = np.concatenate([ql.reshape(T, H, L), P.download(b["d_q_rope_out"], x, (T, H, RP))], -1)
        return m, q, out

    last = rng.standard_normal((R, V))  # the logits behind each request's last token
    for n in range(6):
        lens = [len(h) for h in hist]
        adds = [int(v) for v in rng.integers(1, 14, R)]
        if n == 3:  # request 2 ends; its pages go back
            hist[2], lens[2], adds[2] = [], 0, 0
        parent = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(a)] for a in adds] + [[]]).astype(np.int32)
        kv = P.as_type(rng.standard_normal((sum(adds), W)), x)
        m, q, out = step(lens, adds, parent, kv)
        slot, pos, mask = m.get("slot"), m.get("pos"), m.get("mask")
        rows = cached(slot)
        with np.errstate(invalid="ignore"):
            code, e = S.quantise(P.latent_row(kv, norm, eps, L, pos, theta)[:, :L])
        assert np.array_equal(rows[:, :L], S.values(code, e))
        t = 0
        token, row, start = rng.integers(0, V, sum(adds)), [], []
        for r, a in enumerate(adds):
            keys = np.array(hist[r] + list(rows[t:t + a])).reshape(-1, W)
            for i in range(a):
                seen = S.window_seen(int(mask[t + i]), i, lens[r], a, window, sinks)
                y, far = S.attention(q[t + i], keys, L, scale, seen, x, True)
                assert np.all(np.abs(out[t + i] - y) <= far)
                row.append(t + parent[t + i] if parent[t + i] >= 0 else sum(adds) + r)
            start.append(t)
            t += a
        # the nodes' logits, and those behind the requests' last tokens: each drafted token by its parent's
        z = np.concatenate([out.reshape(len(out), -1).astype(np.float64) @ head, last])
        p = S.Logprobs(z, x, token, row, n_top=4).run()
        p.check()
        logp = p.get("logp", len(token))
        accepted = []
        for r, a in enumerate(adds):  # the likeliest node's path, and what would come behind it
            tip = start[r] + int(np.argmax(logp[start[r]:start[r] + a])) if a else -1
            path = [j for j in range(a) if int(mask[tip]) >> j & 1] if a else []
            accepted.append([start[r] + j for j in path])
            if a:
                last[r] = z[tip]
        src = [j for path in accepted for j in path]
        step(lens, [len(path) for path in accepted], np.concatenate([np.arange(len(path)) - 1 for path in accepted]).astype(np.int32),
             kv, src=src)
        for r, path in enumerate(accepted):
            hist[r] += list(rows[path])
    counts = [len(h) for h in hist]
    got, status = P.upload(np.zeros((sum(counts), W)), "f32"), i32([0])
    b = dict(d_table=i32(table), d_cu=i32(np.concatenate([[0], np.cumsum(counts)])))
    paged.read_rows(paged.RowRead(cache=c, dtype=0, n_req=R, n_rows=sum(counts), max_pages=max_pages, d_out=got.ptr, out_stride=W,
                                  d_status=status.ptr, **{k: v.ptr for k, v in b.items()}))
    hip.synchronize()
    assert status.download(np.int32)[0] == 0
    assert np.array_equal(P.download(got, "f32", (sum(counts), W)), np.concatenate([np.array(h).reshape(-1, W) for h in hist]))


def test_calls_on_streams_and_in_graphs(gpu):
    """The calls on a stream beside others on another; then captured, each graph with its own scratch, and replayed among
    eager calls: the same bits every time."""
    lens, adds = [900, 5, 64], [9, 1, 17]

    def tree(seed, q, cache, window):
        masks = random_trees(np.random.default_rng(seed), adds)
        return S.Serving(seed, q, cache, 512, 64, 16, 64, lens, adds, masks, window=window, sinks=2).upload()
    calls = [tree(20, "bf16", "mxfp4", 0), tree(21, "f32", "mxfp4", 100), tree(22, "bf16", "bf16", 100), tree(23, "f32", "f32", 33)]
    rng = np.random.default_rng(7)
    logp = S.Logprobs(2.5 * rng.standard_normal((27, 20000)), "bf16", rng.integers(0, 20000, 50), rng.integers(0, 27, 50), n_top=7)
    w = Write(6, 300, "f32", 256, 32, 20, 32)
    rows = i32([0] * (300 * 288))
    table = i32(w.slot[:1] // 32)
    read = paged.RowRead(cache=w.c, dtype=0, n_req=1, n_rows=300, max_pages=1, d_table=table.ptr, d_cu=i32([0, 32]).ptr, d_out=rows.ptr,
                         out_stride=288)
    cu = i32([0, 32])
    read.d_cu = cu.ptr
    s1, s2 = hip.Stream(), hip.Stream()

    def others(s):
        paged.token_logprobs(logp.args, s)
        paged.write_rows(w.args, s)
        paged.read_rows(read, s)
    for _ in range(5):
        for t in calls[:2]:
            t.call(s1.handle)
        for t in calls[2:]:
            t.call(s2.handle)
        others(s2.handle)
    hip.synchronize()
    for t in calls:
        t.check()
    first, first_rows = [t.out() for t in calls], rows.download(np.int32)
    graphs = []
    for t in calls:
        g = hip.Graph(s1)
        g.begin()
        t.call(s1.handle)
        g.end()
        graphs.append(g)
    g = hip.Graph(s2)
    g.begin()
    others(s2.handle)
    g.end()
    graphs.append(g)
    for k in range(4):
        for t in calls:
            t.b["d_out"].upload(np.zeros(t.b["d_out"].nbytes, np.uint8))
        rows.upload(np.zeros(rows.nbytes, np.uint8))
        for name in ("d_logp", "d_entropy", "d_top_logp", "d_top_id"):
            logp.b[name].upload(np.zeros(logp.b[name].nbytes - 4, np.uint8))
        for g in graphs:
            g.launch()
        hip.synchronize()
        for t, want in zip(calls, first):
            assert np.array_equal(t.out(), want)
        logp.check()
        w.check()
        assert np.array_equal(rows.download(np.int32), first_rows)
        calls[k].call()  # eager work between the replays
        others(None)
        hip.synchronize()
        assert np.array_equal(calls[k].out(), first[k])
    for g in graphs:
        g.destroy()
    s1.destroy()
    s2.destroy()
