"""What the paged-cache calls refuse on the host, before anything is enqueued
(no device is used: the addresses are never looked at)."""
import ctypes

import pytest

from windlass_amd import moe, paged

BASE = 1 << 40


def at(i):
    return BASE + (i << 32)


def a_map(**change):
    f = dict(n_req=4, page_size=16, n_pages=100, max_pages=8, max_tokens=50)
    for i, n in enumerate(["d_len", "d_add", "d_have", "d_free", "d_n_free", "d_parent", "d_table", "d_have_out",
                           "d_n_free_out", "d_cu", "d_slot", "d_pos", "d_mask", "d_status"]):
        f[n] = at(i)
    return paged.PageMap(**{**f, **change})


def a_cache(**change):
    return paged.Cache(**{**dict(d_rows=at(20), dtype=1, n_pages=100, page_size=16, kv_lora_rank=512, qk_rope=64,
                                 row_stride=576), **change})


def a_write(cache=None, **change):
    f = dict(cache=cache or a_cache(), dtype=0, n_tokens=5, n_heads=4, eps=1e-6, rope_theta=1e4, kv_stride=576, q_stride=256,
             q_out_stride=256)
    for i, n in enumerate(["d_kv", "d_norm_w", "d_pos", "d_slot", "d_q_rope", "d_q_rope_out"]):
        f[n] = at(i)
    return paged.RowWrite(**{**f, **change})


def a_tree(cache=None, **change):
    f = dict(cache=cache or a_cache(), dtype=0, n_req=4, n_tokens=9, n_heads=4, max_pages=8, scale=0.1, q_lat_stride=2048,
             q_rope_stride=256, out_stride=2048, scratch_bytes=1 << 30)
    for i, n in enumerate(["d_q_lat", "d_q_rope", "d_out", "d_table", "d_len", "d_cu", "d_mask", "d_scratch"]):
        f[n] = at(i)
    return paged.TreeAttention(**{**f, **change})


def refused(call, args):
    with pytest.raises(moe.WindlassError) as e:
        call(args)
    assert e.value.status == 1 and len(str(e.value)) > len("WL_ERR_INVALID: wl_paged_map: ")


@pytest.mark.parametrize("change", [
    dict(n_req=4097), dict(page_size=0), dict(page_size=4), dict(page_size=24), dict(page_size=2048), dict(n_pages=0), dict(n_pages=1 << 27),
    dict(max_pages=0), dict(max_pages=1 << 29), dict(max_tokens=1 << 30), dict(d_len=None), dict(d_free=None),
    dict(d_n_free=None), dict(d_table=None), dict(d_cu=None), dict(d_slot=None), dict(d_len=at(0) + 2), dict(d_mask=at(12) + 4),
    dict(d_have_out=at(2)), dict(d_n_free_out=at(4)), dict(d_slot=at(5)), dict(d_pos=at(10) + 196), dict(d_table=at(3) + 396)],
    ids=str)
def test_map_refuses(change):
    refused(paged.page_map, a_map(**change))


CACHES = [dict(d_rows=None), dict(d_rows=at(20) + 8), dict(dtype=2), dict(n_pages=0), dict(n_pages=1 << 27), dict(page_size=48), dict(page_size=4),
          dict(kv_lora_rank=0), dict(kv_lora_rank=516), dict(kv_lora_rank=520, row_stride=640), dict(qk_rope=4),
          dict(qk_rope=72, row_stride=640), dict(qk_rope=0), dict(row_stride=568), dict(row_stride=580)]


@pytest.mark.parametrize("change", CACHES, ids=str)
def test_caches_refused(change):
    refused(paged.write_rows, a_write(a_cache(**change)))
    refused(paged.tree_attention, a_tree(a_cache(**change)))
    refused(paged.tree_attention_scratch, a_tree(a_cache(**change)))


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(n_heads=1025), dict(n_tokens=(1 << 24) + 1), dict(rope_theta=0.0), dict(rope_theta=float("nan")),
    dict(eps=-1.0), dict(eps=float("nan")), dict(d_kv=None), dict(d_kv=at(0) + 8), dict(kv_stride=568), dict(kv_stride=580),
    dict(d_norm_w=None), dict(d_norm_w=at(1) + 2), dict(d_pos=None), dict(d_slot=at(3) + 1), dict(d_q_rope=None),
    dict(q_stride=248), dict(q_out_stride=257), dict(d_q_rope_out=at(4) + 16), dict(d_q_rope_out=at(4), q_out_stride=512),
    dict(d_kv=at(20)), dict(d_q_rope_out=at(0) + 64)], ids=str)
def test_write_refuses(change):
    refused(paged.write_rows, a_write(**change))


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(n_req=4097), dict(n_heads=0), dict(n_heads=1025), dict(n_tokens=(1 << 20) + 1), dict(max_pages=0),
    dict(max_pages=1 << 27), dict(d_q_lat=None), dict(d_q_lat=at(0) + 4), dict(q_lat_stride=2040), dict(q_rope_stride=260),
    dict(d_out=None), dict(out_stride=2044), dict(d_table=None), dict(d_len=None), dict(d_cu=at(5) + 2), dict(d_mask=at(6) + 4),
    dict(d_scratch=None), dict(d_scratch=at(7) + 8), dict(scratch_bytes=0), dict(d_out=at(0)), dict(d_out=at(20) + 160),
    dict(d_scratch=at(2))], ids=str)
def test_tree_attention_refuses(change):
    refused(paged.tree_attention, a_tree(**change))


def test_f32_caches_need_f32_queries():
    refused(paged.tree_attention, a_tree(a_cache(dtype=0), dtype=1))


def test_nothing_to_do_needs_no_device():
    paged.write_rows(a_write(n_tokens=0, d_kv=None))
    paged.tree_attention(a_tree(n_req=0))
    paged.tree_attention(a_tree(n_tokens=0))


def test_null_blocks():
    lib = paged._load()
    for fn in (lib.wl_paged_map, lib.wl_paged_write, lib.wl_paged_tree_attention):
        assert fn(None, None) == 1
    assert lib.wl_paged_tree_scratch(None) == 0
    assert lib.wl_paged_last_error()


def test_argument_blocks_are_laid_out_as_the_header_has_them(tmp_path):
    """Sizes and offsets of the binding's structures against the C compiler's."""
    import os
    import re
    import subprocess
    blocks = {"wl_paged_cache": paged.Cache, "wl_page_map": paged.PageMap, "wl_row_write": paged.RowWrite,
              "wl_tree_attn": paged.TreeAttention}
    lines = []
    for name, cls in blocks.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text("#include <stdio.h>\n#include \"windlass_moe.h\"\nint main(void){" + "".join(lines) + "return 0;}")
    inc = os.path.join(os.path.dirname(moe.HEADER))
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(tmp_path / "s")], check=True)
    got = dict(re.findall(r"(\S+) (\d+)", subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout))
    for name, cls in blocks.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for f in cls._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(cls, f[0]).offset
