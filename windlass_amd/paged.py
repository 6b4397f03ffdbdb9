"""ctypes binding of the paged-cache calls of include/windlass_moe.h: the page
map, the write of latent cache rows and their reading back, attention for trees of
drafted tokens, through a sliding window too, and their log probabilities.

An argument block is one of the structures below, its pointers device
addresses; a program fills it once and passes it to every call whose buffers
stay the same. Marshalling only, as windlass_amd.moe."""
import ctypes

from . import moe

TYPE = {"f32": 0, "bf16": 1, "mxfp4": 4}  # (mxfp4: of a cache's rows)
MAX_REQ = 4096
TREE_MAX_NODES = 64
LOGPROB_MAX_TOP = 32
E_LEN, E_SPACE, E_PAGE, E_TREE, E_SLOT = 1, 2, 4, 8, 16

_vp, _u32, _u64, _f32 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_float


class Cache(ctypes.Structure):
    """wl_paged_cache"""
    _fields_ = [("d_rows", _vp), ("dtype", _u32), ("n_pages", _u32), ("page_size", _u32), ("kv_lora_rank", _u32),
                ("qk_rope", _u32), ("row_stride", _u32)]


class PageMap(ctypes.Structure):
    """wl_page_map"""
    _fields_ = [(n, _u32) for n in ["n_req", "page_size", "n_pages", "max_pages", "max_tokens"]] + \
               [(n, _vp) for n in ["d_len", "d_add", "d_have", "d_free", "d_n_free", "d_parent", "d_table",
                                   "d_have_out", "d_n_free_out", "d_cu", "d_slot", "d_pos", "d_mask", "d_status"]]


class RowWrite(ctypes.Structure):
    """wl_row_write"""
    _fields_ = [("cache", Cache), ("dtype", _u32), ("n_tokens", _u32), ("n_heads", _u32), ("eps", _f32),
                ("rope_theta", _f32), ("d_kv", _vp), ("kv_stride", _u64), ("d_norm_w", _vp), ("d_pos", _vp),
                ("d_slot", _vp), ("d_src", _vp), ("n_kv", _u32), ("d_q_rope", _vp), ("q_stride", _u64),
                ("d_q_rope_out", _vp), ("q_out_stride", _u64), ("d_status", _vp)]


class TreeAttention(ctypes.Structure):
    """wl_tree_attn"""
    _fields_ = [("cache", Cache), ("dtype", _u32), ("n_req", _u32), ("n_tokens", _u32), ("n_heads", _u32),
                ("max_pages", _u32), ("scale", _f32), ("d_q_lat", _vp), ("q_lat_stride", _u64), ("d_q_rope", _vp),
                ("q_rope_stride", _u64), ("d_out", _vp), ("out_stride", _u64), ("d_table", _vp), ("d_len", _vp),
                ("d_cu", _vp), ("d_mask", _vp), ("d_scratch", _vp), ("scratch_bytes", ctypes.c_size_t),
                ("d_status", _vp)]


class WindowAttention(ctypes.Structure):
    """wl_window_attn"""
    _fields_ = [("tree", TreeAttention), ("window", _u32), ("n_sinks", _u32)]


class RowRead(ctypes.Structure):
    """wl_row_read"""
    _fields_ = [("cache", Cache), ("dtype", _u32), ("n_req", _u32), ("n_rows", _u32), ("max_pages", _u32),
                ("d_table", _vp), ("d_first", _vp), ("d_cu", _vp), ("d_out", _vp), ("out_stride", _u64),
                ("d_status", _vp)]


class TokenLogprobs(ctypes.Structure):
    """wl_logprobs"""
    _fields_ = [(n, _u32) for n in ["dtype", "n_rows", "n_vocab", "n_tokens", "n_top"]] + \
               [("d_logits", _vp), ("stride", _u64), ("d_token", _vp), ("d_row", _vp), ("d_logp", _vp),
                ("d_entropy", _vp), ("d_top_logp", _vp), ("d_top_id", _vp), ("d_scratch", _vp),
                ("scratch_bytes", ctypes.c_size_t), ("d_status", _vp)]


_lib = None


def _load():
    global _lib
    if _lib is None:
        lib = moe.load()
        for name, block in [("wl_paged_map", PageMap), ("wl_paged_write", RowWrite),
                            ("wl_paged_tree_attention", TreeAttention), ("wl_paged_window_attention", WindowAttention),
                            ("wl_paged_read", RowRead), ("wl_token_logprobs", TokenLogprobs)]:
            fn = getattr(lib, name)
            fn.argtypes = [ctypes.POINTER(block), _vp]
            fn.restype = ctypes.c_int
        lib.wl_paged_tree_scratch.argtypes = [ctypes.POINTER(TreeAttention)]
        lib.wl_paged_tree_scratch.restype = ctypes.c_size_t
        lib.wl_token_logprobs_scratch.argtypes = [ctypes.POINTER(TokenLogprobs)]
        lib.wl_token_logprobs_scratch.restype = ctypes.c_size_t
        lib.wl_paged_last_error.argtypes = []
        lib.wl_paged_last_error.restype = ctypes.c_char_p
        _lib = lib
    return _lib


def _ck(rc, what):
    if rc != moe.WL_OK:
        raise moe.WindlassError(rc, f"{what}: {_lib.wl_paged_last_error().decode()}")


def page_map(args, stream=0):
    _ck(_load().wl_paged_map(args, stream), "wl_paged_map")


def write_rows(args, stream=0):
    _ck(_load().wl_paged_write(args, stream), "wl_paged_write")


def tree_attention(args, stream=0):
    _ck(_load().wl_paged_tree_attention(args, stream), "wl_paged_tree_attention")


def window_attention(args, stream=0):
    _ck(_load().wl_paged_window_attention(args, stream), "wl_paged_window_attention")


def read_rows(args, stream=0):
    _ck(_load().wl_paged_read(args, stream), "wl_paged_read")


def token_logprobs(args, stream=0):
    _ck(_load().wl_token_logprobs(args, stream), "wl_token_logprobs")


def token_logprobs_scratch(args):
    """Bytes of scratch that token_logprobs needs for these shapes (raises if they are invalid)."""
    n = _load().wl_token_logprobs_scratch(args)
    if n == 0:
        raise moe.WindlassError(1, f"wl_token_logprobs_scratch: {_lib.wl_paged_last_error().decode()}")
    return n


def tree_attention_scratch(args):
    """Bytes of scratch that tree_attention needs for these shapes (raises if they are invalid)."""
    n = _load().wl_paged_tree_scratch(args)
    if n == 0:
        raise moe.WindlassError(1, f"wl_paged_tree_scratch: {_lib.wl_paged_last_error().decode()}")
    return n
