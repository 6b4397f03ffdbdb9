"""The paged-cache operators as timed cases: the page map, the write of latent
cache rows, and attention for trees of drafted tokens over them.

A serving loop that verifies drafted tokens makes these calls each step: one
map of the step's requests (block tables, cache slots, positions and ancestor
masks, from the requests' lengths), then for every layer one write of the new
tokens' rows and one attention of all their heads over the paged cache of
latent rows (a compressed row of kv_lora_rank values, which is key and value at
once, and a rotated key of qk_rope values beside it).

Kinds of cases:

  map    wl_paged_map
  write  wl_paged_write
  attn   wl_paged_tree_attention

run() computes the same outputs in elementary torch operations where `own` is
false, and through the library's binding where it is true; exact() computes
them once more in 64 bits, request by request. Requests' lengths are a case's
own, their order and all values the seed's.
"""
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
THETA = 1e6
NOPE = 192  # the part of a head's dimension that the latent row stands for (the scores' scale)
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _attn(name, n_req, nodes, keys, q="bf16", cache="bf16", heads=64, lora=512, rope=64, page=64, tree=True):
    return dict(name=name, kind="attn", n_req=n_req, nodes=nodes, keys=keys, q=q, cache=cache, heads=heads, lora=lora,
                rope=rope, page=page, tree=tree)


def _write(name, tokens, x, cache, heads=64, lora=512, rope=64, page=64):
    return dict(name=name, kind="write", tokens=tokens, x=x, cache=cache, heads=heads, lora=lora, rope=rope, page=page)


def listed():
    return [
        # a few chats, each with a small tree of drafted tokens: the smallest call
        dict(name="map_8", kind="map", n_req=8, add=8, keys=4096, page=64, tree=True),
        # a full serving batch with the largest trees, long contexts, small pages
        dict(name="map_256", kind="map", n_req=256, add=64, keys=32768, page=16, tree=True),
        # many prompts taken up in one step: no trees, every page new
        dict(name="map_prompts", kind="map", n_req=1000, add=2048, keys=4096, page=32, tree=False),
        # one token of one chat: its row, and its heads' rotary queries
        _write("write_1", 1, "f32", "bf16"),
        # the trees of a serving batch in 32 bits, as a program that keeps the decode's own precision holds them
        _write("write_333", 333, "f32", "f32"),
        # a long prompt, everything in 16 bits
        _write("write_16384", 16384, "bf16", "bf16"),
        # one token of one chat
        _attn("attn_1x1", 1, 1, 4096, tree=False),
        # a batch of chats decoding one token each, long and uneven contexts
        _attn("attn_32x1", 32, 1, 65536, tree=False),
        # the largest tree over one context, 32-bit queries
        _attn("attn_1x64", 1, 64, 8192, q="f32"),
        # a few small trees in 32 bits throughout, the precision of the one-position attention
        _attn("attn_5x7", 5, 7, 2000, q="f32", cache="f32", page=16),
        # a serving batch verifying its drafts
        _attn("attn_64x8", 64, 8, 8192),
        # a smaller model: few heads, a narrow latent row, odd counts
        _attn("attn_12x5", 12, 5, 3001, q="f32", heads=20, lora=256, rope=32, page=32),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], uniform over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    most = {"map": listed()[2], "write": listed()[5], "attn": listed()[10]}
    most = {k: work(c) for k, c in most.items()}
    while True:
        r = rng.random()
        page = rng.choice([16, 32, 64, 128])
        model = dict(heads=rng.choice([64, 64, 64, 128, 32, 20, 16, 8]), lora=512, rope=64)
        if rng.random() < 0.3:
            model.update(lora=8 * rng.randint(12, 64), rope=8 * rng.randint(2, 8))
        if r < 0.2:
            tree = rng.random() < 0.6
            c = dict(kind="map", n_req=_log(rng, 1, 1000), add=_log(rng, 1, 64 if tree else 2048),
                     keys=_log(rng, 16, 32768), page=page, tree=tree)
        elif r < 0.4:
            x, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
            c = dict(kind="write", tokens=_log(rng, 1, 16384), x=x, cache=cache, page=page, **model)
        else:
            q, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
            nodes = 1 if rng.random() < 0.3 else _log(rng, 2, 64)
            c = dict(kind="attn", n_req=_log(rng, 1, 64), nodes=nodes, keys=_log(rng, 16, 65536), q=q, cache=cache,
                     page=page, tree=nodes > 1 and rng.random() < 0.8, **model)
            # the products of 32-bit values cost several of 16-bit ones, and the
            # plain form pads every request to the longest
            w = work(c)
            if w["flops"] * (1 if q == "bf16" else 3 if cache == "bf16" else 6) > most["attn"]["flops"]:
                continue
            if c["n_req"] * c["nodes"] * c["heads"] * c["keys"] > 64 * 8 * 64 * 8192 or c["n_req"] * c["keys"] > 32 * 65536:
                continue
        if work(c)["bytes"] <= most[c["kind"]]["bytes"]:
            return c


# ---- a case's requests --------------------------------------------------------
def _spread(c, what, n, lo, hi):
    """n sizes of [lo, hi], uniform over the logarithm, the first of them hi: the case's own."""
    rng = random.Random(repr((what, sorted((k, v) for k, v in c.items() if k != "name"))))
    return [hi] + [_log(rng, lo, hi) for _ in range(n - 1)]


def _requests(c):
    """(tokens in the cache, tokens added) of every request. In a map case one request of sixteen has ended: it adds
    nothing and gives its pages back."""
    R = c["n_req"]
    if c["kind"] == "attn":
        return _spread(c, "len", R, max(1, c["keys"] // 16), c["keys"]), _spread(c, "add", R, max(1, c["nodes"] // 4), c["nodes"])
    lens = _spread(c, "len", R, max(1, c["keys"] // 16), c["keys"])
    adds = _spread(c, "add", R, max(1, c["add"] // 16), c["add"])
    if not c["tree"]:
        lens = [n if r % 8 == 7 else 0 for r, n in enumerate(lens)]  # most are new, some go on with a long prompt
    for r in range(15, R, 16):
        lens[r] = adds[r] = 0
    return lens, adds


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
    i = torch.cat([torch.arange(a, device=DEV) for a in add]) if add else torch.zeros(0, device=DEV)
    return (torch.rand(len(i), generator=g, device=DEV) * (i + 1)).floor().clamp_max(i).int() - 1


def _ancestors(parent, add):
    """(64-bit masks of a node and its ancestors, depths), by pointer doubling over all trees at once."""
    start = torch.repeat_interleave(torch.cumsum(add, 0) - add, add, output_size=len(parent))
    i = torch.arange(len(parent), device=DEV) - start
    mask = torch.bitwise_left_shift(torch.ones_like(i), i)
    up = torch.where(parent >= 0, parent + start, -1)
    depth = (parent >= 0).long()
    for _ in range(6):
        has = up >= 0
        at = up.clamp_min(0)
        mask = torch.where(has, mask | mask[at], mask)
        depth = torch.where(has, depth + depth[at], depth)
        up = torch.where(has, up[at], -1)
    return mask, depth


def _p(t):
    return None if t is None else t.data_ptr()


def _cache(paged, s, c):
    """The binding's description of the case's cache."""
    return paged.Cache(d_rows=_p(s.cache), dtype=paged.TYPE[c["cache"]], n_pages=s.cache.shape[0], page_size=c["page"],
                       kv_lora_rank=c["lora"], qk_rope=c["rope"], row_stride=c["lora"] + c["rope"])


class _State:
    """What a program holds: its buffers, and the calls' argument blocks that name them."""

    def __init__(self, case):
        self.case = case


def prepare(case, seed):
    s = _State(case)
    {"map": _prepare_map, "write": _prepare_write, "attn": _prepare_attn}[case["kind"]](s, case, seed)
    torch.cuda.synchronize()
    return s


def _prepare_map(s, c, seed):
    R, ps = c["n_req"], c["page"]
    lens, adds = _requests(c)
    # some requests still hold pages of drafts that were turned down, ended ones all they had
    have = [-(-n // ps) + (r % 3 if n else 0) if a else max(1, c["keys"] // ps) for r, (n, a) in enumerate(zip(lens, adds))]
    order = list(range(R))
    random.Random(seed).shuffle(order)
    lens, adds, have = [lens[r] for r in order], [adds[r] for r in order], [have[r] for r in order]
    s.max_pages = max(max(have), max(-(-(n + a) // ps) for n, a in zip(lens, adds)))
    s.n_tokens = sum(adds)
    new = sum(max(0, -(-(n + a) // ps) - h) for n, a, h in zip(lens, adds, have))
    n_free = new + 64
    s.n_pages = sum(have) + n_free
    pages = torch.randperm(s.n_pages, generator=_gen(seed, 1), device=DEV).int()
    s.len, s.add, s.have = _i32(lens), _i32(adds), _i32(have)
    s.table = torch.full((R, s.max_pages), -1, dtype=torch.int32, device=DEV)
    held = torch.arange(s.max_pages, device=DEV) < s.have[:, None]
    s.table[held] = pages[n_free:]
    s.free = torch.full((s.n_pages,), -1, dtype=torch.int32, device=DEV)
    s.free[:n_free] = pages[:n_free]
    s.n_free = _i32([n_free])
    s.parent = _parents(_gen(seed, 2), adds) if c["tree"] else None
    s.have_out, s.n_free_out, s.cu = torch.empty_like(s.have), torch.empty_like(s.n_free), _i32([0] * (R + 1))
    s.slot = torch.empty(s.n_tokens, dtype=torch.int32, device=DEV)
    s.pos = torch.empty_like(s.slot)
    s.mask = torch.empty(s.n_tokens, dtype=torch.int64, device=DEV) if c["tree"] else None
    s.status = _i32([0])
    if own:
        from windlass_amd import paged
        s.args = paged.PageMap(n_req=R, page_size=ps, n_pages=s.n_pages, max_pages=s.max_pages, max_tokens=s.n_tokens,
                               d_len=_p(s.len), d_add=_p(s.add), d_have=_p(s.have), d_free=_p(s.free),
                               d_n_free=_p(s.n_free), d_parent=_p(s.parent), d_table=_p(s.table),
                               d_have_out=_p(s.have_out), d_n_free_out=_p(s.n_free_out), d_cu=_p(s.cu),
                               d_slot=_p(s.slot), d_pos=_p(s.pos), d_mask=_p(s.mask), d_status=_p(s.status))


def _prepare_write(s, c, seed):
    T, W = c["tokens"], c["lora"] + c["rope"]
    n_pages = -(-T // c["page"]) + 8
    g = _gen(seed, 3)
    s.kv = _randn(g, T, W).to(DTYPE[c["x"]])
    s.q = _randn(g, T, c["heads"], c["rope"]).to(DTYPE[c["x"]])
    s.ln = (1.0 + _randn(g, c["lora"], std=0.1)).to(torch.bfloat16)
    s.pos = torch.randint(0, 1 << 17, (T,), generator=g, device=DEV).int()
    s.slot = torch.randperm(n_pages * c["page"], generator=g, device=DEV)[:T].int()
    s.cache = torch.zeros(n_pages, c["page"], W, dtype=DTYPE[c["cache"]], device=DEV)
    s.q_out = torch.empty_like(s.q)
    s.status = _i32([0])
    if own:
        from windlass_amd import paged
        s.args = paged.RowWrite(cache=_cache(paged, s, c), dtype=paged.TYPE[c["x"]], n_tokens=T, n_heads=c["heads"],
                                eps=EPS, rope_theta=THETA, d_kv=_p(s.kv), kv_stride=W, d_norm_w=_p(s.ln),
                                d_pos=_p(s.pos), d_slot=_p(s.slot), d_q_rope=_p(s.q), q_stride=c["heads"] * c["rope"],
                                d_q_rope_out=_p(s.q_out), q_out_stride=c["heads"] * c["rope"], d_status=_p(s.status))


def _prepare_attn(s, c, seed):
    R, ps, L, W = c["n_req"], c["page"], c["lora"], c["lora"] + c["rope"]
    lens, adds = _requests(c)
    order = list(range(R))
    random.Random(seed).shuffle(order)
    lens, adds = [lens[r] for r in order], [adds[r] for r in order]
    g = _gen(seed, 4)
    held = [-(-(n + a) // ps) for n, a in zip(lens, adds)]
    s.n_tokens, s.max_keys, s.max_nodes = sum(adds), max(n + a for n, a in zip(lens, adds)), max(adds)
    pages = torch.randperm(sum(held) + 4, generator=g, device=DEV).int()
    s.table = torch.zeros(R, max(held), dtype=torch.int32, device=DEV)
    s.table[torch.arange(max(held), device=DEV) < _i32(held)[:, None]] = pages[:sum(held)]
    s.cache = torch.empty(len(pages), ps, W, dtype=DTYPE[c["cache"]], device=DEV).normal_(generator=g)
    s.scale = (NOPE + c["rope"]) ** -0.5
    s.q_lat = _randn(g, s.n_tokens, c["heads"], L, std=2.0 / (s.scale * W ** 0.5)).to(DTYPE[c["q"]])
    s.q_rope = _randn(g, s.n_tokens, c["heads"], c["rope"], std=2.0 / (s.scale * W ** 0.5)).to(DTYPE[c["q"]])
    s.len, s.add = _i32(lens), _i32(adds)
    s.cu = _i32([sum(adds[:r]) for r in range(R + 1)])
    s.mask = _ancestors(_parents(g, adds).long(), s.add.long())[0] if c["tree"] else None
    s.out = torch.empty_like(s.q_lat)
    s.status = _i32([0])
    if own:
        from windlass_amd import paged
        s.args = paged.TreeAttention(cache=_cache(paged, s, c), dtype=paged.TYPE[c["q"]], n_req=R, n_tokens=s.n_tokens,
                                     n_heads=c["heads"], max_pages=max(held), scale=s.scale, d_q_lat=_p(s.q_lat),
                                     q_lat_stride=c["heads"] * L, d_q_rope=_p(s.q_rope),
                                     q_rope_stride=c["heads"] * c["rope"], d_out=_p(s.out), out_stride=c["heads"] * L,
                                     d_table=_p(s.table), d_len=_p(s.len), d_cu=_p(s.cu), d_mask=_p(s.mask),
                                     d_status=_p(s.status))
        s.scratch = torch.empty(paged.tree_attention_scratch(s.args), dtype=torch.uint8, device=DEV)
        s.args.d_scratch, s.args.scratch_bytes = _p(s.scratch), s.scratch.numel()


# ---- one pass -----------------------------------------------------------------
def run(s):
    kind = s.case["kind"]
    if own:
        from windlass_amd import paged
        stream = torch.cuda.current_stream().cuda_stream
        {"map": paged.page_map, "write": paged.write_rows, "attn": paged.tree_attention}[kind](s.args, stream)
    else:
        {"map": _plain_map, "write": _plain_write, "attn": _plain_attn}[kind](s)
    if kind == "map":
        return {"table": s.table, "free": s.free, "have": s.have_out, "n_free": s.n_free_out, "cu": s.cu, "slot": s.slot,
                "pos": s.pos, "mask": s.mask}
    return {"cache": s.cache, "q": s.q_out} if kind == "write" else s.out


def _plain_map(s):
    ps = s.case["page"]
    n, a, h = s.len.long(), s.add.long(), s.have.long()
    need = (n + a + ps - 1) // ps
    col = torch.arange(s.max_pages, device=DEV)
    # surplus pages go on the stack, request by request
    back = (col >= need[:, None]) & (col < h[:, None])
    top = s.n_free + back.sum()
    flat = back.reshape(-1)
    at = s.n_free + torch.cumsum(flat, 0) - 1
    at = torch.where(flat, at, s.n_pages)
    stack = torch.cat([s.free, s.free[:1]])
    stack.scatter_(0, at, s.table.reshape(-1))
    s.free.copy_(stack[:-1])
    # new pages come from its top, request by request
    take = (col >= h[:, None]) & (col < need[:, None])
    k = (torch.cumsum(take.reshape(-1), 0) - 1).view_as(take)
    s.table.copy_(torch.where(take, s.free[(top - 1 - k).clamp_min(0)], s.table))
    s.have_out.copy_(need)
    s.n_free_out.copy_(top - take.sum())
    # the tokens
    cu = torch.cumsum(a, 0)
    s.cu[1:] = cu
    req = torch.repeat_interleave(torch.arange(len(a), device=DEV), a, output_size=s.n_tokens)
    row = torch.arange(s.n_tokens, device=DEV) - (cu - a)[req] + n[req]
    s.slot.copy_(s.table[req, row // ps] * ps + row % ps)
    if s.mask is None:
        s.pos.copy_(row)
    else:
        mask, depth = _ancestors(s.parent.long(), a)
        s.mask.copy_(mask)
        s.pos.copy_(n[req] + depth)


def _rotate(x, pos):
    """Adjacent pairs turned by their angle at `pos` [tokens, ...]; the result holds the halves apart. Angles in 64 bits."""
    n = x.shape[-1]
    inv = THETA ** (-torch.arange(0, n, 2, dtype=torch.float64, device=DEV) / n)
    ang = pos[..., None].double() * inv
    cos, sin = ang.cos().to(x.dtype), ang.sin().to(x.dtype)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_write(s):
    L = s.case["lora"]
    x = s.kv.float()
    c = x[:, :L]
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * s.ln.float()
    row = torch.cat([c, _rotate(x[:, L:], s.pos)], -1)
    s.cache.view(-1, row.shape[-1])[s.slot.long()] = row.to(s.cache.dtype)
    s.q_out.copy_(_rotate(s.q.float(), s.pos[:, None]))


def _plain_attn(s):
    c = s.case
    R, N, K, H, L, ps = c["n_req"], s.max_nodes, s.max_keys, c["heads"], c["lora"], c["page"]
    key = torch.arange(K, device=DEV)
    node = torch.arange(N, device=DEV)
    n, a = s.len.long()[:, None], s.add.long()[:, None]
    # every request padded to the longest: its keys, its queries, what each node sees
    rows = s.table.long()[:, key // ps] * ps + key % ps
    kv = s.cache.view(-1, s.cache.shape[-1])[rows].float()
    at = (s.cu[:-1].long()[:, None] + node).clamp_max(s.n_tokens - 1)
    q = torch.cat([s.q_lat[at], s.q_rope[at]], -1).float().view(R, N * H, -1)
    bits = s.mask[at] if s.mask is not None else (torch.bitwise_left_shift(2, node) - 1).expand(R, N)
    j = (key - n)[:, None, :]
    seen = (j < 0) | (((bits[..., None] >> j.clamp(0, 63)) & 1 == 1) & (j < a[..., None]))
    score = torch.matmul(q, kv.transpose(1, 2)).mul_(s.scale).view(R, N, H, K)
    score.masked_fill_(~seen[:, :, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(R, N * H, K), kv[..., :L]).view(R, N, H, L).div_(total)
    req = torch.repeat_interleave(torch.arange(R, device=DEV), s.add.long(), output_size=s.n_tokens)
    s.out.copy_(out[req, torch.arange(s.n_tokens, device=DEV) - s.cu[req]])


# ---- what a pass cannot do without ---------------------------------------------
_SIZE = {"f32": 4, "bf16": 2}


def work(case):
    c = case
    if c["kind"] == "map":
        lens, adds = _requests(c)
        tokens, ps = sum(adds), c["page"]
        new = sum(-(-(n + a) // ps) - -(-n // ps) for n, a in zip(lens, adds))
        return {"bytes": 20 * c["n_req"] + 8 * new + tokens * (20 if c["tree"] else 8), "flops": 0}
    L, W, H = c["lora"], c["lora"] + c["rope"], c["heads"]
    if c["kind"] == "write":
        T, x = c["tokens"], _SIZE[c["x"]]
        return {"bytes": T * (W * (x + _SIZE[c["cache"]]) + 2 * H * c["rope"] * x + 8) + 2 * L,
                "flops": T * (4 * L + 3 * (H + 1) * c["rope"])}
    lens, adds = _requests(c)
    pairs = sum(n * a for n, a in zip(lens, adds))
    tokens, keys = sum(adds), sum(lens) + sum(adds)
    return {"bytes": keys * W * _SIZE[c["cache"]] + tokens * H * (W + L) * _SIZE[c["q"]] + 4 * (keys // c["page"]),
            "flops": 2 * H * (W + L) * (pairs + tokens)}


# ---- the same in 64 bits --------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"map": _exact_map, "write": _exact_write, "attn": _exact_attn}[case["kind"]](s)


def _exact_map(s):
    """Whole numbers, one request after another."""
    ps, lens, adds, have = s.case["page"], s.len.tolist(), s.add.tolist(), s.have.tolist()
    table, n_free = s.table.tolist(), s.n_free.item()
    stack = s.free.tolist()
    need = [-(-(n + a) // ps) for n, a in zip(lens, adds)]
    for r, h in enumerate(have):
        for k in range(need[r], h):
            stack[n_free] = table[r][k]
            n_free += 1
    cu, slot, pos, mask = [0], [], [], []
    parent = s.parent.tolist() if s.parent is not None else None
    for r, (n, a, h) in enumerate(zip(lens, adds, have)):
        for k in range(h, need[r]):
            n_free -= 1
            table[r][k] = stack[n_free]
        for i in range(a):
            slot.append(table[r][(n + i) // ps] * ps + (n + i) % ps)
            if parent is None:
                pos.append(n + i)
                continue
            p = parent[cu[-1] + i]
            mask.append((1 << i) | (mask[cu[-1] + p] if p >= 0 else 0))
            pos.append(pos[cu[-1] + p] + 1 if p >= 0 else n)
        cu.append(cu[-1] + a)
    mask = [m - (1 << 64) if m >> 63 else m for m in mask]
    return {"table": _i32(table), "free": _i32(stack), "have": _i32(need), "n_free": _i32([n_free]), "cu": _i32(cu),
            "slot": _i32(slot), "pos": _i32(pos),
            "mask": None if parent is None else torch.tensor(mask, dtype=torch.int64, device=DEV)}


def _turn(x, pos):
    """The rotation as a product of complex numbers."""
    half = x.shape[-1] // 2
    ang = pos.double()[:, None] * torch.exp(torch.arange(half, dtype=torch.float64, device=DEV) * (-2.0 / x.shape[-1])
                                            * torch.log(torch.tensor(THETA, dtype=torch.float64, device=DEV)))
    turn = torch.polar(torch.ones_like(ang), ang)
    z = torch.view_as_complex(x.double().unflatten(-1, (half, 2)).contiguous())
    z = z * (turn[:, None] if z.dim() == 3 else turn)
    return torch.cat([z.real, z.imag], -1)


def _exact_write(s):
    L = s.case["lora"]
    x = s.kv.double()
    size = torch.linalg.vector_norm(x[:, :L], dim=-1, keepdim=True)
    c = x[:, :L] / torch.sqrt(size ** 2 / L + EPS) * s.ln.double()
    cache = torch.zeros(s.cache.shape, dtype=torch.float64, device=DEV)
    cache.flatten(0, 1).index_copy_(0, s.slot.long(), torch.cat([c, _turn(x[:, L:], s.pos)], -1))
    return {"cache": cache, "q": _turn(s.q, s.pos)}


def _exact_attn(s):
    c = s.case
    L, ps, flat = c["lora"], c["page"], s.cache.flatten(0, 1)
    out = torch.empty(s.out.shape, dtype=torch.float64, device=DEV)
    lens, adds, cu = s.len.tolist(), s.add.tolist(), s.cu.tolist()
    for r, (n, a) in enumerate(zip(lens, adds)):
        page = s.table[r, :-(-(n + a) // ps)].long()
        kv = flat[(page[:, None] * ps + torch.arange(ps, device=DEV)).reshape(-1)[:n + a]].double()
        for i in range(a):
            t = cu[r] + i
            if s.mask is None:
                see = kv[:n + i + 1]
            else:
                bits = s.mask[t].item()
                tree = [n + j for j in range(a) if bits >> j & 1]
                see = kv if len(tree) == a else torch.cat([kv[:n], kv[tree]])
            q = torch.cat([s.q_lat[t], s.q_rope[t]], -1).double()
            out[t] = torch.softmax(q @ see.T * s.scale, -1) @ see[:, :L]
    return out
