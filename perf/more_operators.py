"""More operators of a serving step as timed cases: the paged cache of latent
rows held in 4 bits, attention through a sliding window with sinks, and the log
probabilities that the verification of drafted tokens reads.

A step of a serving loop over a paged cache writes the new tokens' rows, attends
to the cache for every layer, and scores the drafted tokens by the model's
logits. Here the cache holds its compressed part in MXFP4 (blocks of 32 E2M1
values under one power of two) and the rotated key in bf16: 400 bytes a token
instead of 1152 at 512 + 64 columns.

Kinds of cases:

  rows   wl_paged_write into a 4-bit cache, then wl_paged_read of the same tokens
         (the rows of a request in order, as values: what a prefix is multiplied
         with kv_b_proj from)
  attn   wl_paged_tree_attention over a 4-bit cache (window 0), or
         wl_paged_window_attention over any cache
  logp   wl_token_logprobs

run() computes the same outputs in elementary torch operations where `own` is
false, and through the library's binding where it is true; exact() computes
them once more in 64 bits. Requests' lengths are a case's own, their order and
all values the seed's.
"""
import random

import torch

own = False

DEV = "cuda"
EPS = 2.0 ** -20
THETA = 1e6
NOPE = 192  # the part of a head's dimension that the latent row stands for (the scores' scale)
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
SCALE_LO, SCALE_HI = 2, 252  # the block scales' biased exponents


def _rows(name, n_req, add, keys, x, heads=64, lora=512, rope=64, page=64):
    return dict(name=name, kind="rows", n_req=n_req, add=add, keys=keys, x=x, heads=heads, lora=lora, rope=rope, page=page)


def _attn(name, n_req, nodes, keys, q="bf16", cache="mxfp4", window=0, sinks=0, heads=64, lora=512, rope=64, page=64,
          tree=True):
    return dict(name=name, kind="attn", n_req=n_req, nodes=nodes, keys=keys, q=q, cache=cache, window=window, sinks=sinks,
                heads=heads, lora=lora, rope=rope, page=page, tree=tree)


def _logp(name, rows, vocab, x, per, top):
    return dict(name=name, kind="logp", rows=rows, vocab=vocab, x=x, per=per, top=top)


def listed():
    return [
        # one token of one chat: its row and its heads' rotary queries, and the row read back
        _rows("rows_1", 1, 1, 4096, "f32"),
        # a few long prompts taken up in one step
        _rows("rows_prompts", 5, 4096, 4096, "bf16"),
        # one token of one chat over a 4-bit cache
        _attn("attn4_1x1", 1, 1, 4096, tree=False),
        # a batch of chats decoding one token each, long and uneven contexts
        _attn("attn4_32x1", 32, 1, 65536, tree=False),
        # a serving batch verifying its drafts
        _attn("attn4_64x8", 64, 8, 8192),
        # a few small trees, 32-bit queries over the 4-bit cache
        _attn("attn4_5x7_f32", 5, 7, 2000, q="f32", page=16),
        # the batch of chats again, through a window with sinks
        _attn("win4_32x1", 32, 1, 65536, window=4096, sinks=4, tree=False),
        # drafts of a serving batch through a window, the cache in 16 bits
        _attn("win_64x8", 64, 8, 32768, cache="bf16", window=2048, sinks=64),
        # a smaller model in 32 bits throughout: few heads, a narrow latent row, odd counts
        _attn("win_12x5_f32", 12, 5, 3001, q="f32", cache="f32", window=509, sinks=7, heads=20, lora=256, rope=32, page=32),
        # one token's logits: its log probability and a few alternatives
        _logp("logp_1", 1, 154880, "bf16", 1, 5),
        # the drafts of a serving batch, each scored by its parent's row, the next tokens among 20 alternatives
        _logp("logp_284", 284, 154880, "bf16", 2, 20),
        # a prompt's tokens scored, 32-bit logits of an odd vocabulary, some of it masked
        _logp("logp_1024_f32", 1024, 100003, "f32", 1, 0),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    top = {c["name"]: work(c) for c in listed()}
    while True:
        r = rng.random()
        page = rng.choice([16, 32, 64, 128])
        model = dict(heads=rng.choice([64, 64, 64, 128, 32, 20, 16, 8]), lora=512, rope=64)
        if rng.random() < 0.3:
            model.update(lora=32 * rng.randint(3, 16), rope=8 * rng.randint(2, 8))
        if r < 0.2:
            c = dict(kind="rows", n_req=_log(rng, 1, 64), add=_log(rng, 1, 4096), keys=_log(rng, 16, 8192),
                     x=rng.choice(["f32", "bf16"]), page=page, **model)
            if work(c)["bytes"] <= top["rows_prompts"]["bytes"]:
                return c
        elif r < 0.75:
            q, cache = rng.choice([("bf16", "mxfp4"), ("bf16", "mxfp4"), ("f32", "mxfp4"), ("bf16", "bf16"), ("f32", "bf16"),
                                   ("f32", "f32")])
            nodes = 1 if rng.random() < 0.3 else _log(rng, 2, 64)
            window = 0 if cache == "mxfp4" and rng.random() < 0.5 else _log(rng, 1, 8192)
            c = dict(kind="attn", n_req=_log(rng, 1, 64), nodes=nodes, keys=_log(rng, 16, 65536), q=q, cache=cache,
                     window=window, sinks=0 if window == 0 or rng.random() < 0.3 else _log(rng, 1, 128), page=page,
                     tree=nodes > 1 and rng.random() < 0.8, **model)
            # the products of 32-bit values cost several of 16-bit ones, and the
            # plain form pads every request to the longest
            w = work(c)
            if w["flops"] * (1 if q == "bf16" else 6 if cache == "f32" else 3) > top["attn4_64x8"]["flops"]:
                continue
            if w["bytes"] > top["attn4_32x1"]["bytes"]:
                continue
            keys = min(c["keys"], window + c["sinks"]) if window else c["keys"]
            if c["n_req"] * c["nodes"] * c["heads"] * keys <= 64 * 8 * 64 * 8192 and c["n_req"] * keys <= 32 * 65536 and \
               c["n_req"] * c["keys"] <= 64 * 32768:
                return c
        else:
            c = dict(kind="logp", rows=_log(rng, 1, 2048), vocab=_log(rng, 1000, 160000), x=rng.choice(["f32", "bf16"]),
                     per=rng.choice([1, 1, 2, 3]), top=rng.choice([0, 1, 5, 20, 32]))
            if work(c)["bytes"] <= top["logp_1024_f32"]["bytes"]:
                return c


# ---- a case's requests --------------------------------------------------------
def _spread(c, what, n, lo, hi):
    """n sizes of [lo, hi], uniform over the logarithm, the first of them hi: the case's own."""
    rng = random.Random(repr((what, sorted((k, v) for k, v in c.items() if k != "name"))))
    return [hi] + [_log(rng, lo, hi) for _ in range(n - 1)]


def _requests(c):
    """(tokens in the cache, tokens added) of every request."""
    R = c["n_req"]
    n = c["add"] if c["kind"] == "rows" else c["nodes"]
    return _spread(c, "len", R, max(1, c["keys"] // 16), c["keys"]), _spread(c, "add", R, max(1, n // 4), n)


def _gen(seed, *tags):
    g = torch.Generator(device=DEV)
    s = seed
    for t in tags:
        s = (s * 1000003 + t + 1) & 0x7FFFFFFFFFFF
    g.manual_seed(s)
    return g


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _parents(g, add):
    """Parents of the nodes of trees of add[r] nodes, in a row: -1 or an earlier node of the same tree."""
    i = torch.cat([torch.arange(a, device=DEV) for a in add])
    return (torch.rand(len(i), generator=g, device=DEV) * (i + 1)).floor().clamp_max(i).int() - 1


def _ancestors(parent, add):
    """64-bit masks of a node and its ancestors, by pointer doubling over all trees at once."""
    start = torch.repeat_interleave(torch.cumsum(add, 0) - add, add, output_size=len(parent))
    i = torch.arange(len(parent), device=DEV) - start
    mask = torch.bitwise_left_shift(torch.ones_like(i), i)
    up = torch.where(parent >= 0, parent + start, -1)
    for _ in range(6):
        has = up >= 0
        at = up.clamp_min(0)
        mask = torch.where(has, mask | mask[at], mask)
        up = torch.where(has, up[at], -1)
    return mask


def _p(t):
    return None if t is None else t.data_ptr()


def _row_bytes(c):
    """Bytes of a row of a 4-bit cache: nibbles, 16 bytes of block scales, the rotated key in bf16."""
    return c["lora"] // 2 + 16 + 2 * c["rope"]


def _cache(paged, s, c, dtype):
    """The binding's description of the case's cache."""
    mx = dtype == "mxfp4"
    return paged.Cache(d_rows=_p(s.cache), dtype=paged.TYPE[dtype], n_pages=s.cache.shape[0], page_size=c["page"],
                       kv_lora_rank=c["lora"], qk_rope=c["rope"], row_stride=_row_bytes(c) if mx else c["lora"] + c["rope"])


class _State:
    """What a program holds: its buffers, and the calls' argument blocks that name them."""

    def __init__(self, case):
        self.case = case


def prepare(case, seed):
    s = _State(case)
    {"rows": _prepare_rows, "attn": _prepare_attn, "logp": _prepare_logp}[case["kind"]](s, case, seed)
    torch.cuda.synchronize()
    return s


def _tables(s, c, g, lens, adds):
    R, ps = c["n_req"], c["page"]
    held = [-(-(n + a) // ps) for n, a in zip(lens, adds)]
    pages = torch.randperm(sum(held) + 4, generator=g, device=DEV).int()
    s.table = torch.zeros(R, max(held), dtype=torch.int32, device=DEV)
    s.table[torch.arange(max(held), device=DEV) < _i32(held)[:, None]] = pages[:sum(held)]
    s.n_tokens = sum(adds)
    s.len, s.add = _i32(lens), _i32(adds)
    s.cu = _i32([sum(adds[:r]) for r in range(R + 1)])
    return len(pages)


def _order(c, seed):
    lens, adds = _requests(c)
    order = list(range(c["n_req"]))
    random.Random(seed).shuffle(order)
    return [lens[r] for r in order], [adds[r] for r in order]


def _prepare_rows(s, c, seed):
    W, H = c["lora"] + c["rope"], c["heads"]
    g = _gen(seed, 3)
    lens, adds = _order(c, seed)
    n_pages = _tables(s, c, g, lens, adds)
    T = s.n_tokens
    s.kv = _randn(g, T, W).to(DTYPE[c["x"]])
    s.q = _randn(g, T, H, c["rope"]).to(DTYPE[c["x"]])
    s.ln = (1.0 + _randn(g, c["lora"], std=0.1)).to(torch.bfloat16)
    req = torch.repeat_interleave(torch.arange(c["n_req"], device=DEV), s.add.long(), output_size=T)
    at = torch.arange(T, device=DEV) - s.cu[req] + s.len[req]
    s.pos = at.int()
    s.slot = (s.table[req, at // c["page"]] * c["page"] + at % c["page"]).int()
    s.cache = torch.zeros(n_pages, c["page"], _row_bytes(c), dtype=torch.uint8, device=DEV)
    s.q_out = torch.empty_like(s.q)
    s.rows = torch.empty(T, W, dtype=torch.bfloat16, device=DEV)
    s.status = _i32([0])
    if own:
        from windlass_amd import paged
        cache = _cache(paged, s, c, "mxfp4")
        s.args = paged.RowWrite(cache=cache, dtype=paged.TYPE[c["x"]], n_tokens=T, n_heads=H, eps=EPS, rope_theta=THETA,
                                d_kv=_p(s.kv), kv_stride=W, d_norm_w=_p(s.ln), d_pos=_p(s.pos), d_slot=_p(s.slot),
                                d_q_rope=_p(s.q), q_stride=H * c["rope"], d_q_rope_out=_p(s.q_out),
                                q_out_stride=H * c["rope"], d_status=_p(s.status))
        s.read = paged.RowRead(cache=cache, dtype=paged.TYPE["bf16"], n_req=c["n_req"], n_rows=T,
                               max_pages=s.table.shape[1], d_table=_p(s.table), d_first=_p(s.len), d_cu=_p(s.cu),
                               d_out=_p(s.rows), out_stride=W, d_status=_p(s.status))


def _prepare_attn(s, c, seed):
    L, W = c["lora"], c["lora"] + c["rope"]
    lens, adds = _order(c, seed)
    g = _gen(seed, 4)
    n_pages = _tables(s, c, g, lens, adds)
    s.max_keys, s.max_nodes = max(n + a for n, a in zip(lens, adds)), max(adds)
    if c["cache"] == "mxfp4":  # rows as the write leaves them: normal values, quantised
        s.cache = torch.empty(n_pages, c["page"], _row_bytes(c), dtype=torch.uint8, device=DEV)
        x = torch.empty(4096 * 1024 // W // c["page"] + 1, c["page"], W, device=DEV)
        for i in range(0, n_pages, len(x)):
            part = s.cache[i:i + len(x)]
            part.copy_(_pack(x.normal_(generator=g)[:len(part)].float(), L))
    else:
        s.cache = torch.empty(n_pages, c["page"], W, dtype=DTYPE[c["cache"]], device=DEV).normal_(generator=g)
    s.scale = (NOPE + c["rope"]) ** -0.5
    s.q_lat = _randn(g, s.n_tokens, c["heads"], L, std=2.0 / (s.scale * W ** 0.5)).to(DTYPE[c["q"]])
    s.q_rope = _randn(g, s.n_tokens, c["heads"], c["rope"], std=2.0 / (s.scale * W ** 0.5)).to(DTYPE[c["q"]])
    s.mask = _ancestors(_parents(g, adds).long(), s.add.long()) if c["tree"] else None
    s.out = torch.empty_like(s.q_lat)
    s.status = _i32([0])
    if own:
        from windlass_amd import paged
        s.args = paged.TreeAttention(cache=_cache(paged, s, c, c["cache"]), dtype=paged.TYPE[c["q"]], n_req=c["n_req"],
                                     n_tokens=s.n_tokens, n_heads=c["heads"], max_pages=s.table.shape[1], scale=s.scale,
                                     d_q_lat=_p(s.q_lat), q_lat_stride=c["heads"] * L, d_q_rope=_p(s.q_rope),
                                     q_rope_stride=c["heads"] * c["rope"], d_out=_p(s.out), out_stride=c["heads"] * L,
                                     d_table=_p(s.table), d_len=_p(s.len), d_cu=_p(s.cu), d_mask=_p(s.mask),
                                     d_status=_p(s.status))
        s.scratch = torch.empty(paged.tree_attention_scratch(s.args), dtype=torch.uint8, device=DEV)
        s.args.d_scratch, s.args.scratch_bytes = _p(s.scratch), s.scratch.numel()
        if c["window"]:
            s.args = paged.WindowAttention(tree=s.args, window=c["window"], n_sinks=c["sinks"])


def _prepare_logp(s, c, seed):
    R, V = c["rows"], c["vocab"]
    g = _gen(seed, 5)
    s.logits = torch.empty(R, V, dtype=DTYPE[c["x"]], device=DEV).normal_(0.0, 2.5, generator=g)
    # a few likely tokens a row, and ids behind the tokenizer's last that may not come
    s.logits.scatter_add_(1, torch.randint(0, V, (R, 8), generator=g, device=DEV),
                          (_randn(g, R, 8, std=3.0) + 10.0).to(s.logits.dtype))
    s.logits[:, V - min(64, V // 16):] = float("-inf")
    s.n_tokens = R * c["per"]
    s.token = torch.randint(0, V - min(64, V // 16), (s.n_tokens,), generator=g, device=DEV).int()
    s.row = torch.randint(0, R, (s.n_tokens,), generator=g, device=DEV).int() if c["per"] > 1 else None
    s.logp = torch.empty(s.n_tokens, device=DEV)
    s.entropy = torch.empty(R, device=DEV)
    s.top_logp = torch.empty(R, c["top"], device=DEV)
    s.top_id = torch.empty(R, c["top"], dtype=torch.int32, device=DEV)
    s.status = _i32([0])
    if own:
        from windlass_amd import paged
        s.args = paged.TokenLogprobs(dtype=paged.TYPE[c["x"]], n_rows=R, n_vocab=V, n_tokens=s.n_tokens, n_top=c["top"],
                                     d_logits=_p(s.logits), stride=V, d_token=_p(s.token), d_row=_p(s.row),
                                     d_logp=_p(s.logp), d_entropy=_p(s.entropy),
                                     d_top_logp=_p(s.top_logp) if c["top"] else None,
                                     d_top_id=_p(s.top_id) if c["top"] else None, d_status=_p(s.status))
        s.scratch = torch.empty(paged.token_logprobs_scratch(s.args), dtype=torch.uint8, device=DEV)
        s.args.d_scratch, s.args.scratch_bytes = _p(s.scratch), s.scratch.numel()


# ---- one pass -----------------------------------------------------------------
def run(s):
    c = s.case
    if own:
        from windlass_amd import paged
        stream = torch.cuda.current_stream().cuda_stream
        if c["kind"] == "rows":
            paged.write_rows(s.args, stream)
            paged.read_rows(s.read, stream)
        elif c["kind"] == "attn":
            (paged.window_attention if c["window"] else paged.tree_attention)(s.args, stream)
        else:
            paged.token_logprobs(s.args, stream)
    else:
        {"rows": _plain_rows, "attn": _plain_attn, "logp": _plain_logp}[c["kind"]](s)
    if c["kind"] == "rows":
        return {"rows": s.rows, "q": s.q_out}
    if c["kind"] == "attn":
        return s.out
    return {"logp": s.logp, "entropy": s.entropy, **({"top_logp": s.top_logp, "top_id": s.top_id} if c["top"] else {})}


def _power(e):
    """2^e for whole numbers e of [-126, 127], exactly."""
    return (e.int() + 127 << 23).view(torch.float32)


def _quantise(x):
    """x [..., 32 n] in 64 bits -> (E2M1 codes with signs, biased exponents [..., n]). A block's exponent is the least with
    which its largest magnitude is at most 6; values go to the nearest of E2M1, the even code where two are as near."""
    b = x.unflatten(-1, (-1, 32))
    size = b.abs().amax(-1)
    m, e = torch.frexp(size)  # size = m 2^e, m in [1/2, 1): at most 6 = 0.75 2^3 from e - 3 on, or one more
    e = torch.where(size > 0, e - 3 + (m > 0.75), -1000).clamp(SCALE_LO - 127, SCALE_HI - 127)
    a = b.abs() * _power(-e[..., None])
    code = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return torch.where(torch.signbit(b) & (code > 0), code + 8, code).flatten(-2), e + 127


def _value(code, exponent):
    """The values that codes and biased exponents stand for, in 32 bits."""
    lut = torch.tensor(E2M1 + [-v for v in E2M1], device=DEV)
    return (lut[code.int()].unflatten(-1, (-1, 32)) * _power(exponent.int()[..., None] - 127)).flatten(-2)


def _scale_at(n):
    """Where a row's scale bytes stand: block b's at 4 (b % 4) + b / 4."""
    b = torch.arange(n, device=DEV)
    return 4 * (b % 4) + b // 4


def _pack(x, L):
    """Rows of a 4-bit cache for values x [..., W]."""
    code, e = _quantise(x[..., :L])
    scales = torch.zeros(*x.shape[:-1], 16, dtype=torch.uint8, device=DEV)
    scales[..., _scale_at(L // 32)] = e.byte()
    rope = x[..., L:].to(torch.bfloat16).contiguous().view(torch.uint8)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, scales, rope], -1)


def _unpack(rows, L):
    """The values (32 bits) of rows of a 4-bit cache."""
    n = rows[..., :L // 2]
    code = torch.stack([n & 15, n >> 4], -1).flatten(-2)
    rope = rows[..., L // 2 + 16:].contiguous().view(torch.bfloat16).float()
    return torch.cat([_value(code, rows[..., L // 2:L // 2 + 16][..., _scale_at(L // 32)]), rope], -1)


def _rotate(x, pos):
    """Adjacent pairs turned by their angle at `pos` [tokens, ...]; the result holds the halves apart. Angles in 64 bits."""
    n = x.shape[-1]
    inv = THETA ** (-torch.arange(0, n, 2, dtype=torch.float64, device=DEV) / n)
    ang = pos[..., None].double() * inv
    cos, sin = ang.cos().to(x.dtype), ang.sin().to(x.dtype)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_rows(s):
    L = s.case["lora"]
    x = s.kv.double()  # values next to a border of 4-bit ones
    c = x[:, :L]
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s.ln.double()
    row = _rotate(x[:, L:].float(), s.pos)
    s.cache.view(-1, s.cache.shape[-1])[s.slot.long()] = _pack(torch.cat([c, row], -1), L)
    s.q_out.copy_(_rotate(s.q.float(), s.pos[:, None]))
    s.rows.copy_(_unpack(s.cache.view(-1, s.cache.shape[-1])[s.slot.long()], L))


def _plain_attn(s):
    c = s.case
    R, N, H, L, ps, win, sinks = c["n_req"], s.max_nodes, c["heads"], c["lora"], c["page"], c["window"], c["sinks"]
    node = torch.arange(N, device=DEV)
    n, a = s.len.long()[:, None], s.add.long()[:, None]
    # every request padded to the longest: its keys that some node may see, its queries, what each node sees
    if win and sinks + win + N < s.max_keys:
        first = (n - win + 1).clamp_min(sinks)  # behind the sinks
        key = torch.cat([torch.arange(sinks, device=DEV).expand(R, -1), first + torch.arange(win + N, device=DEV)], 1)
    else:
        key = torch.arange(s.max_keys, device=DEV).expand(R, -1)
    K = key.shape[1]
    held = key < n + a
    at = torch.where(held, key, 0)
    rows = torch.gather(s.table.long(), 1, at // ps) * ps + at % ps
    kv = s.cache.view(-1, s.cache.shape[-1])[rows]
    kv = _unpack(kv, L) if c["cache"] == "mxfp4" else kv.float()
    at = (s.cu[:-1].long()[:, None] + node).clamp_max(s.n_tokens - 1)
    q = torch.cat([s.q_lat[at], s.q_rope[at]], -1).float().view(R, N * H, -1)
    bits = s.mask[at] if s.mask is not None else (torch.bitwise_left_shift(2, node) - 1).expand(R, N)
    j = (key - n)[:, None, :]
    in_tree = (bits[..., None] >> j.clamp(0, 63)) & 1 == 1
    seen = held[:, None, :] & ((j < 0) | in_tree)
    if win:  # positions: a node's is the number of its ancestors behind the request's tokens
        up = (bits[..., None] >> node) & 1  # [R, N, ancestors]
        depth = torch.where(node < node[:, None], up, 0).sum(-1)
        rank = torch.cumsum(up, -1) - up  # of an ancestor among them
        kpos = torch.where(j < 0, key[:, None, :], n[..., None] + rank.gather(2, j.clamp(0, N - 1).expand(R, N, K)))
        seen &= (kpos < sinks) | ((n + depth)[..., None] - kpos < win)
    score = torch.matmul(q, kv.transpose(1, 2)).mul_(s.scale).view(R, N, H, K)
    score.masked_fill_(~seen[:, :, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(R, N * H, K), kv[..., :L]).view(R, N, H, L).div_(total)
    req = torch.repeat_interleave(torch.arange(R, device=DEV), s.add.long(), output_size=s.n_tokens)
    s.out.copy_(out[req, torch.arange(s.n_tokens, device=DEV) - s.cu[req]])


def _plain_logp(s):
    z = s.logits.float() + 0.0
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(-1, keepdim=True)
    lse = top + total.log()
    row = torch.arange(len(z), device=DEV) if s.row is None else s.row.long()
    s.logp.copy_(z[row, s.token.long()] - lse[row, 0])
    s.entropy.copy_((total.log() - (e * (z - top).clamp_min(-1e30)).sum(-1, keepdim=True) / total)[:, 0])
    k = s.case["top"]
    if k:  # the largest, of equal ones the lowest id: in the order of (value, -id) as one integer
        i = z.view(torch.int32)
        i = torch.where(i < 0, i ^ 0x7FFFFFFF, i).long()
        order = (i << 32) + (z.shape[1] - 1 - torch.arange(z.shape[1], device=DEV))
        best = torch.topk(order, k, -1).values
        s.top_id.copy_(z.shape[1] - 1 - (best & 0xFFFFFFFF))
        s.top_logp.copy_(z.gather(1, s.top_id.long()) - lse)


# ---- what a pass cannot do without ---------------------------------------------
_SIZE = {"f32": 4, "bf16": 2}


def _cache_bytes(c, dtype):
    """Bytes of a row, without padding."""
    return c["lora"] // 2 + c["lora"] // 32 + 2 * c["rope"] if dtype == "mxfp4" else (c["lora"] + c["rope"]) * _SIZE[dtype]


def work(case):
    c = case
    if c["kind"] == "logp":
        R, V = c["rows"], c["vocab"]
        return {"bytes": R * V * _SIZE[c["x"]] + R * c["per"] * 12 + R * (4 + 8 * c["top"]), "flops": 4 * R * V}
    L, W, H = c["lora"], c["lora"] + c["rope"], c["heads"]
    lens, adds = _requests(c)
    tokens = sum(adds)
    if c["kind"] == "rows":
        x = _SIZE[c["x"]]
        return {"bytes": tokens * (W * (x + 2) + 2 * _cache_bytes(c, "mxfp4") + 2 * H * c["rope"] * x + 8) + 2 * L,
                "flops": tokens * (5 * L + 3 * (H + 1) * c["rope"])}
    if c["window"]:
        lens = [min(n, c["window"] + c["sinks"]) for n in lens]
    pairs = sum(n * a for n, a in zip(lens, adds))
    keys = sum(lens) + tokens
    return {"bytes": keys * _cache_bytes(c, c["cache"]) + tokens * H * (W + L) * _SIZE[c["q"]] + 4 * (keys // c["page"]),
            "flops": 2 * H * (W + L) * (pairs + tokens)}


# ---- the same in 64 bits --------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"rows": _exact_rows, "attn": _exact_attn, "logp": _exact_logp}[case["kind"]](s)


def _turn(x, pos):
    """The rotation as a product of complex numbers."""
    half = x.shape[-1] // 2
    ang = pos.double()[:, None] * torch.exp(torch.arange(half, dtype=torch.float64, device=DEV) * (-2.0 / x.shape[-1])
                                            * torch.log(torch.tensor(THETA, dtype=torch.float64, device=DEV)))
    turn = torch.polar(torch.ones_like(ang), ang)
    z = torch.view_as_complex(x.double().unflatten(-1, (half, 2)).contiguous())
    z = z * (turn[:, None] if z.dim() == 3 else turn)
    return torch.cat([z.real, z.imag], -1)


def _exact_rows(s):
    """The nearest of the sixteen values to each quotient, by distance."""
    L = s.case["lora"]
    x = s.kv.double()
    size = torch.linalg.vector_norm(x[:, :L], dim=-1, keepdim=True)
    c = (x[:, :L] / torch.sqrt(size ** 2 / L + EPS) * s.ln.double()).view(len(x), -1, 32)
    most = c.abs().amax(-1, keepdim=True)
    unit = torch.full_like(most, 2.0 ** (SCALE_LO - 127))
    for e in range(SCALE_LO - 126, 128):  # (this path's values lie far below the largest scale)
        unit = torch.where(most > 6 * unit, 2.0 ** e, unit)
    grid = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=DEV)  # even codes first
    near = torch.stack([((c.abs() / unit) - v).abs() for v in grid]).argmin(0)
    value = (grid[near] * unit * torch.sign(c)).view(len(x), L)
    return {"rows": torch.cat([value, _turn(x[:, L:], s.pos)], -1), "q": _turn(s.q, s.pos)}


def _exact_values(s, rows):
    """The values of cache rows [k, ...] in 64 bits."""
    c, L = s.case, s.case["lora"]
    if c["cache"] != "mxfp4":
        return rows.double()
    code = torch.empty(len(rows), L, dtype=torch.long, device=DEV)
    code[:, 0::2], code[:, 1::2] = (rows[:, :L // 2] % 16).long(), (rows[:, :L // 2] // 16).long()
    size = torch.where(code % 8 < 2, 0.5 * (code % 8).double(), (1 + 0.5 * (code % 2).double()) * 2.0 ** (code % 8 // 2 - 1))
    for b in range(L // 32):
        size[:, 32 * b:32 * b + 32] *= 2.0 ** (rows[:, L // 2 + 4 * (b % 4) + b // 4].double()[:, None] - 127)
    return torch.cat([torch.where(code >= 8, -size, size), rows[:, L // 2 + 16:].contiguous().view(torch.bfloat16).double()], 1)


def _exact_attn(s):
    c = s.case
    L, ps, win, flat = c["lora"], c["page"], c["window"], s.cache.flatten(0, 1)
    if s.n_tokens * (min(c["keys"], win + c["sinks"]) if win else c["keys"]) > 1 << 23:
        return None  # too long in 64 bits, token by token
    out = torch.empty(s.out.shape, dtype=torch.float64, device=DEV)
    lens, adds, cu = s.len.tolist(), s.add.tolist(), s.cu.tolist()
    for r, (n, a) in enumerate(zip(lens, adds)):
        page = s.table[r, :-(-(n + a) // ps)].long()
        start = max(0, min(n, n - win + 1)) if win else 0
        keys = list(range(min(start, c["sinks"]))) + list(range(start, n + a))
        at = torch.tensor(keys, device=DEV)
        kv = _exact_values(s, flat[page[at // ps] * ps + at % ps])
        for i in range(a):
            t = cu[r] + i
            bits = (2 << i) - 1 if s.mask is None else s.mask[t].item()
            tree = [j for j in range(a) if bits >> j & 1]
            pos = {n + j: n + k for k, j in enumerate(tree)}
            mine = pos[n + i]
            if win:
                see = [k for k, key in enumerate(keys)
                       if (key < n or key in pos) and (pos.get(key, key) < c["sinks"] or mine - pos.get(key, key) < win)]
            else:
                see = list(range(n)) + [n + j for j in tree]
            x = kv[torch.tensor(see, device=DEV)]
            q = torch.cat([s.q_lat[t], s.q_rope[t]], -1).double()
            out[t] = torch.softmax(q @ x.T * s.scale, -1) @ x[:, :L]
    return out


def _exact_logp(s):
    c, k = s.case, s.case["top"]
    row = s.row.long() if s.row is not None else torch.arange(s.n_tokens, device=DEV)
    lse = torch.empty(c["rows"], dtype=torch.float64, device=DEV)
    entropy, picked = torch.empty_like(lse), torch.empty(s.n_tokens, dtype=torch.float64, device=DEV)
    top, ids = torch.empty(c["rows"], k, dtype=torch.float64, device=DEV), torch.empty(c["rows"], k, dtype=torch.int32, device=DEV)
    for a in range(0, c["rows"], 128):
        z = s.logits[a:a + 128].double()
        lse[a:a + 128] = torch.logsumexp(z, -1)
        p = torch.softmax(z, -1)
        entropy[a:a + 128] = torch.special.entr(p).sum(-1)
        col = torch.arange(c["vocab"], device=DEV)
        for j in range(k):  # the largest left, of equal ones the first
            best = z.amax(-1, keepdim=True)
            i = torch.where(z == best, col, c["vocab"]).amin(-1, keepdim=True)
            top[a:a + 128, j:j + 1], ids[a:a + 128, j:j + 1] = best - lse[a:a + 128, None], i.int()
            z.scatter_(1, i, float("-inf"))
    picked = s.logits[row, s.token.long()].double() - lse[row]
    return {"logp": picked, "entropy": entropy, **({"top_logp": top, "top_id": ids} if k else {})}
