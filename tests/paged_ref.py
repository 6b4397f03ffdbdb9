"""Plain 64-bit counterparts of the paged-cache calls, and the buffers of a
call, for tests/test_gpu_paged*.py."""
import numpy as np

from windlass_amd import hip, paged

U32 = 2.0 ** -24  # half a step of f32, bf16
U16 = 2.0 ** -8
E4 = np.dtype(np.float32)


def bf16_bits(x):
    """f32 -> bf16 bits, round to nearest even (NaN kept)."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_value(b):
    return (np.ascontiguousarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def as_type(x, t):
    """The values of x as type t holds them (f32 array)."""
    return bf16_value(bf16_bits(x)) if t == "bf16" else np.ascontiguousarray(x, np.float32)


def upload(x, t):
    return hip.DeviceBuffer.from_array(bf16_bits(x) if t == "bf16" else np.ascontiguousarray(x, np.float32))


def download(buf, t, shape):
    n = int(np.prod(shape))
    return (bf16_value(buf.download(np.uint16, n)) if t == "bf16" else buf.download(np.float32, n)).reshape(shape)


def page_map(ps, max_pages, n_pages, lens, adds, have, free, n_free, table, parent=None):
    """(table, free, have, n_free, cu, slot, pos, mask) after a step that is not refused."""
    table, free = table.copy(), free.copy()
    need = [-(-(n + a) // ps) for n, a in zip(lens, adds)]
    for r, h in enumerate(have):
        for k in range(need[r], h):
            free[n_free] = table[r, k]
            n_free += 1
    cu, slot, pos, mask = [0], [], [], []
    for r, (n, a, h) in enumerate(zip(lens, adds, have)):
        for k in range(h, need[r]):
            n_free -= 1
            table[r, k] = free[n_free]
        depth, bits = [], []
        for i in range(a):
            slot.append(table[r, (n + i) // ps] * ps + (n + i) % ps)
            p = i - 1 if parent is None else int(parent[cu[-1] + i])
            p = p if -1 <= p < i else -1
            depth.append(depth[p] + 1 if p >= 0 else 0)
            bits.append((1 << i) | (bits[p] if p >= 0 else 0))
        pos += [n + d for d in depth]
        mask += bits
        cu.append(cu[-1] + a)
    return table, free, np.array(need), n_free, np.array(cu), np.array(slot), np.array(pos), mask


def rope(x, pos, theta):
    n = x.shape[-1]
    ang = np.asarray(pos, np.float64)[..., None] * theta ** (-np.arange(0, n, 2) / n)
    a, b = x[..., 0::2].astype(np.float64), x[..., 1::2].astype(np.float64)
    return np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)], -1)


def latent_row(kv, w, eps, L, pos, theta):
    c = kv[..., :L].astype(np.float64)
    c = c / np.sqrt((c * c).mean(-1, keepdims=True) + eps) * w
    return np.concatenate([c, rope(kv[..., L:], pos, theta)], -1)


def tree_attention(q, rows, L, scale, seen, q_type):
    """q [H, W], rows [K, W], seen [K] -> (out [H, L], how far a kernel may be off).

    The bound: with u = 2^-24, a score of W products summed in f32 in any order
    is off by at most (W + 16) u scale sum|q k|, and its exponential's argument
    by 4 u |s| more; weights are then off by that much relatively, their sum by
    as much again, and sums over K keys (each key joined, rescaled and added in
    f32) by (K + 64) u; exponentials and the quotient by 16 u. A bf16 output
    adds 2^-8 for its weights' rounding and 2^-8 of itself for its own."""
    H = q.shape[0]
    if not seen.any():
        return np.zeros((H, L)), np.zeros((H, L))
    q, k = q.astype(np.float64), rows[seen].astype(np.float64)
    s = scale * q @ k.T
    es = ((k.shape[1] + 16) * U32 * abs(scale) * (np.abs(q) @ np.abs(k).T) + 4 * U32 * np.abs(s)).max(1, keepdims=True)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    out, size = p @ k[:, :L], p @ np.abs(k[:, :L])
    far = size * np.expm1(2 * es + (len(k) + 80) * U32)
    if q_type == "bf16":
        far = far + U16 * (size + np.abs(out)) * (1 + U16)
    return out, far + 1e-37


def tree_attention_mean(q, rows, L, scale, seen, q_type):
    """tree_attention for results that are means by rounded weights. For a bf16 output: with weights p (1 + d), |d| <=
    2^-8, over their own sum the result is off by sum p d (c - out) / sum p (1 + d), at most 2^-8 / (1 - 2^-8) sum p |c -
    out|, and 2^-8 of itself for its own rounding; f32 sums and exponentials as there."""
    out, far = tree_attention(q, rows, L, scale, seen, "f32")
    if q_type == "bf16" and seen.any():
        k = rows[seen].astype(np.float64)
        s = scale * q.astype(np.float64) @ k.T
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        dev = np.stack([w @ np.abs(k[:, :L] - o) for w, o in zip(p, out)])
        far = (far + U16 / (1 - U16) * dev) * (1 + U16) + U16 * np.abs(out)
    return out, far


class Map:
    """The buffers of a wl_page_map."""

    def __init__(self, ps, n_pages, max_pages, lens, adds, have, free, n_free, table, parent=None, max_tokens=None, trees=None,
                 fill=-7):
        R, T = len(lens), sum(max(a, 0) for a in adds) if max_tokens is None else max_tokens
        i32 = lambda x: hip.DeviceBuffer.from_array(np.asarray(x, np.int32).reshape(-1))  # noqa: E731
        self.R, self.T, self.shape = R, T, (R, max_pages)
        b = self.b = dict(d_len=i32(lens), d_add=i32(adds), d_have=i32(have), d_free=i32(free), d_n_free=i32([n_free]),
                          d_table=i32(table), d_have_out=i32([fill] * R), d_n_free_out=i32([fill]),
                          d_cu=i32([fill] * (R + 1)), d_slot=i32([fill] * T), d_pos=i32([fill] * T), d_status=i32([0]))
        if parent is not None:
            b["d_parent"] = i32(parent)
        if trees if trees is not None else parent is not None:
            b["d_mask"] = hip.DeviceBuffer.from_array(np.full(T, 77, np.uint64))
        self.n_pages = n_pages
        self.args = paged.PageMap(n_req=R, page_size=ps, n_pages=n_pages, max_pages=max_pages, max_tokens=T,
                                  **{k: v.ptr for k, v in b.items()})

    def get(self, name):
        n = {"table": self.R * self.shape[1], "free": self.n_pages, "have_out": self.R, "n_free_out": 1, "cu": self.R + 1,
             "slot": self.T, "pos": self.T, "mask": self.T, "status": 1}[name]
        x = self.b["d_" + name].download(np.uint64 if name == "mask" else np.int32, n)
        return x.reshape(self.shape) if name == "table" else x
