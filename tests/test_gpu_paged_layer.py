"""The paged calls against wl_run_attention: the same layer, its positions one
call each there, a prompt and chains of drafted tokens here (run with -m gpu)."""
import numpy as np
import pytest

from oracle import moe_oracle as O
from oracle import synth
from tests import paged_ref as P
from tests.test_gpu_attention import FCFG, GLM_ATTN, TOL, _step
from windlass_amd import hip, paged, synthdata
from windlass_amd.model import AttnModel

pytestmark = pytest.mark.gpu
TYPE = paged.TYPE["f32"]


@pytest.mark.parametrize("a,steps", [(dict(FCFG, index_topk=64), [7, 1, 5, 12, 1]), (dict(GLM_ATTN, index_topk=2048), [40, 1, 8, 3])],
                         ids=["small", "glm"])
def test_paged_calls_are_the_layers_attention(gpu, a, steps):
    """Up to index_topk keys, where a layer attends to all of them. Projections in 64 bits from the layer's own norm and
    q_a outputs; what stands before o_proj is within the sum of both sides' bars, each TOL of the largest value."""
    H, L, RP, ND, V, ps, n = a["n_heads"], a["kv_lora_rank"], a["qk_rope"], a["qk_nope"], a["v_head"], 16, sum(steps)
    am = AttnModel(a, 3, 1, owners=[True], max_seq=n)
    got = [_step(am, 0, p, synth.hidden_state(a["hidden"], 77, p)) for p in range(n)]
    W = {k: v.astype(np.float64) for k, v in synthdata.as_f32(am.weights[0]).items()}
    norm, qr = (np.stack([g[k] for g in got]).astype(np.float64) for k in ("norm", "q_resid"))
    kv = (norm @ W["kv_a_proj"].T).astype(np.float32)
    q = (qr @ W["q_b_proj"].T).reshape(n, H, ND + RP)
    kv_b = W["kv_b_proj"].reshape(H, ND + V, L)
    q_lat = np.einsum("thd,hdl->thl", q[..., :ND], kv_b[:, :ND]).astype(np.float32)
    q_rope = np.ascontiguousarray(q[..., ND:], np.float32)
    n_pages = -(-n // ps) + 3
    cache = hip.DeviceBuffer.from_array(np.full((n_pages * ps, L + RP), np.nan, np.float32))
    c = paged.Cache(d_rows=cache.ptr, dtype=TYPE, n_pages=n_pages, page_size=ps, kv_lora_rank=L, qk_rope=RP, row_stride=L + RP)
    norm_w = P.upload(W["kv_a_ln"], "bf16")
    at, have, n_free = 0, 0, n_pages
    table, free = np.full((1, n_pages), -1, np.int32), np.random.default_rng(4).permutation(n_pages).astype(np.int32)
    out = []
    for t in steps:
        m = P.Map(ps, n_pages, n_pages, [at], [t], [have], free, n_free, table)
        paged.page_map(m.args)
        b = dict(d_kv=P.upload(kv[at:at + t], "f32"), q=P.upload(q_rope[at:at + t], "f32"), lat=P.upload(q_lat[at:at + t], "f32"),
                 out=hip.DeviceBuffer(4 * t * H * L))
        paged.write_rows(paged.RowWrite(cache=c, dtype=TYPE, n_tokens=t, n_heads=H, eps=1e-6, rope_theta=a["rope_theta"],
                                        d_kv=b["d_kv"].ptr, kv_stride=L + RP, d_norm_w=norm_w.ptr, d_pos=m.b["d_pos"].ptr,
                                        d_slot=m.b["d_slot"].ptr, d_q_rope=b["q"].ptr, q_stride=H * RP,
                                        d_q_rope_out=b["q"].ptr, q_out_stride=H * RP, d_status=m.b["d_status"].ptr))
        x = paged.TreeAttention(cache=c, dtype=TYPE, n_req=1, n_tokens=t, n_heads=H, max_pages=n_pages, scale=(ND + RP) ** -0.5,
                                d_q_lat=b["lat"].ptr, q_lat_stride=H * L, d_q_rope=b["q"].ptr, q_rope_stride=H * RP,
                                d_out=b["out"].ptr, out_stride=H * L, d_table=m.b["d_table"].ptr, d_len=m.b["d_len"].ptr,
                                d_cu=m.b["d_cu"].ptr, d_status=m.b["d_status"].ptr)
        size = paged.tree_attention_scratch(x)
        b["scratch"] = hip.DeviceBuffer(size)
        x.d_scratch, x.scratch_bytes = b["scratch"].ptr, size
        paged.tree_attention(x)
        hip.synchronize()
        assert m.get("status")[0] == 0
        out.append(b["out"].download(np.float32, t * H * L).reshape(t, H, L))
        table, free, n_free, have = m.get("table"), m.get("free"), int(m.get("n_free_out")[0]), int(m.get("have_out")[0])
        at += t
    attn = np.einsum("thl,hvl->thv", np.concatenate(out).astype(np.float64), kv_b[:, ND:]).reshape(n, H * V)
    worst = max(O.rel_to_scale(g["attn"], y) for g, y in zip(got, attn))
    am.close()
    assert worst < 2 * TOL
    print(f"paged calls against run_attention: worst {worst:.2e}", flush=True)
