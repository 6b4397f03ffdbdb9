"""What the calls of the 4-bit cache, the window and the log probabilities refuse on the host, before anything is
enqueued (no device is used: the addresses are never looked at)."""
import ctypes
import os
import re
import subprocess

import pytest

from windlass_amd import moe, paged

from .test_paged_args import a_cache, a_tree, a_write, at, refused


def mx_cache(**change):
    return a_cache(**{**dict(dtype=4, row_stride=400), **change})


def a_window(tree=None, **change):
    return paged.WindowAttention(**{**dict(tree=tree or a_tree(), window=100, n_sinks=4), **change})


def a_read(cache=None, **change):
    f = dict(cache=cache or a_cache(), dtype=0, n_req=4, n_rows=9, max_pages=8, out_stride=576)
    for i, n in enumerate(["d_table", "d_first", "d_cu", "d_out", "d_status"]):
        f[n] = at(i)
    return paged.RowRead(**{**f, **change})


def some_logits(**change):
    f = dict(dtype=0, n_rows=4, n_vocab=1000, n_tokens=4, n_top=5, stride=1000, scratch_bytes=1 << 30)
    for i, n in enumerate(["d_logits", "d_token", "d_logp", "d_entropy", "d_top_logp", "d_top_id", "d_scratch", "d_status"]):
        f[n] = at(i)
    return paged.TokenLogprobs(**{**f, **change})


MX_CACHES = [dict(d_rows=None), dict(d_rows=at(20) + 8), dict(dtype=3), dict(dtype=5), dict(n_pages=0), dict(page_size=4),
             dict(kv_lora_rank=488), dict(kv_lora_rank=0), dict(kv_lora_rank=544, row_stride=640), dict(qk_rope=4),
             dict(qk_rope=72, row_stride=640), dict(row_stride=384), dict(row_stride=408), dict(row_stride=(1 << 21) + 16)]


@pytest.mark.parametrize("change", MX_CACHES, ids=str)
def test_mx_caches_refused(change):
    c = mx_cache(**change)
    refused(paged.write_rows, a_write(c))
    refused(paged.tree_attention, a_tree(c))
    refused(paged.tree_attention, a_tree(c, dtype=1))
    refused(paged.tree_attention_scratch, a_tree(c))
    refused(paged.window_attention, a_window(a_tree(c)))
    refused(paged.read_rows, a_read(c))


def test_mx_is_a_type_of_caches_only():
    refused(paged.write_rows, a_write(dtype=4))
    refused(paged.tree_attention, a_tree(mx_cache(), dtype=4))
    refused(paged.read_rows, a_read(dtype=4))
    refused(paged.token_logprobs, some_logits(dtype=4))


def test_mx_overlaps():
    """A 4-bit cache spans its rows' bytes: 1600 rows of 400."""
    refused(paged.write_rows, a_write(mx_cache(), d_kv=at(20) + 1600 * 400 - 16))
    refused(paged.tree_attention, a_tree(mx_cache(), d_out=at(20) + 1600 * 400 - 16))
    refused(paged.read_rows, a_read(mx_cache(), d_out=at(20) + 1600 * 400 - 16))


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(n_req=4097), dict(n_heads=0), dict(max_pages=0), dict(d_q_lat=None), dict(q_rope_stride=260),
    dict(d_out=None), dict(d_table=None), dict(d_scratch=at(7) + 8), dict(scratch_bytes=0), dict(d_out=at(0)), dict(d_scratch=at(2))],
    ids=str)
def test_window_attention_refuses_what_tree_attention_does(change):
    refused(paged.window_attention, a_window(a_tree(**change)))
    refused(paged.window_attention, a_window(a_tree(**change), window=0))


def test_window_f32_caches_need_f32_queries():
    refused(paged.window_attention, a_window(a_tree(a_cache(dtype=0), dtype=1)))


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(n_req=4097), dict(n_rows=(1 << 24) + 1), dict(max_pages=0), dict(max_pages=1 << 27), dict(d_table=None),
    dict(d_table=at(0) + 2), dict(d_first=at(1) + 1), dict(d_cu=None), dict(d_cu=at(2) + 2), dict(d_out=None), dict(d_out=at(3) + 8),
    dict(out_stride=568), dict(out_stride=580), dict(out_stride=(1 << 22) + 8), dict(d_out=at(20)), dict(d_out=at(0)), dict(d_out=at(2)),
    dict(d_status=at(4) + 2), dict(d_status=at(3) + 16)], ids=str)
def test_read_refuses(change):
    refused(paged.read_rows, a_read(**change))


@pytest.mark.parametrize("change", [
    dict(dtype=2), dict(n_vocab=0), dict(n_vocab=(1 << 20) + 1, stride=1 << 21), dict(n_rows=(1 << 20) + 1), dict(n_tokens=(1 << 20) + 1),
    dict(n_top=33), dict(n_vocab=3, n_top=4), dict(d_logits=None), dict(d_logits=at(0) + 2), dict(stride=999),
    dict(stride=(1 << 24) + 1), dict(d_token=None), dict(d_logp=None), dict(n_tokens=5), dict(n_rows=0), dict(d_top_id=None),
    dict(d_top_logp=None), dict(d_token=at(1) + 2), dict(d_row=at(9) + 1), dict(d_logp=at(2) + 2), dict(d_entropy=at(3) + 1),
    dict(d_status=at(7) + 3), dict(d_scratch=None), dict(d_scratch=at(6) + 8), dict(scratch_bytes=0), dict(d_logp=at(0) + 400),
    dict(d_entropy=at(1)), dict(d_top_id=at(4) + 40), dict(d_logp=at(3)), dict(d_scratch=at(0)), dict(d_entropy=at(6) + 16)], ids=str)
def test_logprobs_refuses(change):
    refused(paged.token_logprobs, some_logits(**change))


def test_logprobs_scratch_refuses():
    refused(paged.token_logprobs_scratch, some_logits(n_vocab=0))
    assert paged.token_logprobs_scratch(some_logits()) % 4 == 0


def test_nothing_to_do_needs_no_device():
    paged.write_rows(a_write(mx_cache(), n_tokens=0, d_kv=None))
    paged.window_attention(a_window(a_tree(n_req=0)))
    paged.window_attention(a_window(a_tree(mx_cache(), n_tokens=0)))
    paged.read_rows(a_read(n_req=0))
    paged.read_rows(a_read(n_rows=0, d_out=None))
    paged.token_logprobs(some_logits(n_rows=0, n_tokens=0, d_logits=None))


def test_null_blocks():
    lib = paged._load()
    for fn in (lib.wl_paged_window_attention, lib.wl_paged_read, lib.wl_token_logprobs):
        assert fn(None, None) == 1
    assert lib.wl_token_logprobs_scratch(None) == 0


def test_argument_blocks_are_laid_out_as_the_header_has_them(tmp_path):
    blocks = {"wl_window_attn": paged.WindowAttention, "wl_row_read": paged.RowRead, "wl_logprobs": paged.TokenLogprobs}
    lines = ['printf("types %d %d %d\\n", WL_TYPE_MXFP4, WL_LOGPROB_MAX_TOP, WL_TYPE_BF16);']
    for name, cls in blocks.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text("#include <stdio.h>\n#include \"windlass_moe.h\"\nint main(void){" + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-I", os.path.dirname(moe.HEADER), str(src), "-o", str(tmp_path / "s")], check=True)
    text = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout
    assert text.startswith(f"types {paged.TYPE['mxfp4']} {paged.LOGPROB_MAX_TOP} {paged.TYPE['bf16']}\n")
    got = dict(re.findall(r"^(\S+) (\d+)$", text, re.M))
    for name, cls in blocks.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for f in cls._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(cls, f[0]).offset


@pytest.mark.parametrize("n_vocab", [1, 1000, 2049, 32000, 154880, 1 << 20])
def test_logprobs_scratch_of_a_batch_is_enough_for_smaller_ones(n_vocab):
    """A program takes it once, for its largest call."""
    def need(rows, vocab, top):
        return paged.token_logprobs_scratch(some_logits(n_rows=rows, n_vocab=vocab, stride=1 << 20, n_top=top))
    most = {}
    for top in {0, 1, min(32, n_vocab)}:
        for rows in [*range(1, 300), 511, 512, 513, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 20000, 1 << 20]:
            n = need(rows, n_vocab, top)
            for fewer in ((rows - 1, n_vocab, top), (rows, n_vocab - 1, min(top, n_vocab - 1)), (rows, n_vocab, 0)):
                if min(fewer[:2]) > 0:
                    assert need(*fewer) <= n, fewer
            most[top] = max(most.get(top, 0), n)
            assert n == most[top]  # in the order of the rows


def test_logprobs_with_the_scratch_of_a_larger_batch():
    """284 rows of a step, 256 of the next: not refused for its scratch (but for what is checked after it)."""
    n = paged.token_logprobs_scratch(some_logits(n_rows=284, n_vocab=154880, stride=154880, n_top=20))
    with pytest.raises(moe.WindlassError, match="overlap"):
        paged.token_logprobs(some_logits(n_rows=256, n_vocab=154880, stride=154880, n_top=20, scratch_bytes=n, d_logp=at(3)))
