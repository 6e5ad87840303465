"""Workloads of the 4-bit KV cache: quantising keys and values into a paged
cache as they are written, reading them back, and attention over the cache.

``run`` computes each operator either in its plain form (elementary torch
operations in 32 bits, rounded once to the output's type) or, with ``own``
set, through the framework's entry points (moe_fused_inference_b200.kv4).

Definition of the cache.  A token's key or value vector of one KV head
(head_dim = 64 or 128) is cut into blocks of 32 elements.  A block with
largest magnitude a is held as an 8-bit exponent code c = e + 127, where e is
the smallest integer >= -99 with 6 * 2^e >= a, and 32 4-bit values: sign and
the nearest of {0, .5, 1, 1.5, 2, 3, 4, 6} to |x| / 2^e, ties to the larger.
A block with a value that is not finite has c = 255 and reads as NaN.

Memory: one uint8 tensor (pages, kv_heads, page / 16, 17 * head_dim).  A tile
of 16 consecutive tokens holds 16 key rows of head_dim / 2 bytes, 16 value
rows, 16 rows of key codes (head_dim / 32 bytes each), 16 rows of value codes.
Even elements sit in a byte's low half.  With nb = head_dim / 32 blocks, the
key row stores the 4-byte word t (8 elements) of block b at word t * nb + b,
the value row the 2-byte piece h (4 elements) of block b at piece h * nb + b.

Token slot s of the pool is token s % page of page s / page.

Attention.  Sequence i owns the query rows cu_q[i] .. cu_q[i + 1] - 1 and the
first kv_lens[i] tokens of the pages page_table[i]; its rows are the last of
these tokens, so row r of R sees the tokens 0 .. kv_lens[i] - R + r, and a row
that sees none gives zeros.  Query head h reads KV head h / (heads / kv_heads).
"""

import math

import torch

own = False

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases --------------------------------------------------------------------
def listed():
    def store(name, tokens, kv_heads, head_dim, page, dtype, fused, padded=0):
        return {"name": name, "op": "store", "tokens": tokens, "kv_heads": kv_heads,
                "head_dim": head_dim, "page": page, "dtype": dtype, "fused": fused,
                "padded": padded}

    def fetch(name, tokens, kv_heads, head_dim, page, dtype):
        return {"name": name, "op": "fetch", "tokens": tokens, "kv_heads": kv_heads,
                "head_dim": head_dim, "page": page, "dtype": dtype}

    def attend(name, seqs, rows, ctx, kv_heads, group, head_dim, page, dtype, fused, hole=False):
        return {"name": name, "op": "attend", "seqs": seqs, "rows_lo": rows[0], "rows_hi": rows[1],
                "ctx_lo": ctx[0], "ctx_hi": ctx[1], "kv_heads": kv_heads, "group": group,
                "head_dim": head_dim, "page": page, "dtype": dtype, "fused": fused, "hole": hole}

    return [
        # one decode step of one sequence: the new token's keys and values
        store("store_token", 1, 4, 128, 64, "bf16", True),
        # odd count of tokens straight from a 32-bit projection, small pages,
        # some rows padding of a captured batch
        store("store_odd", 1021, 2, 64, 16, "fp32", False, padded=13),
        # a long prompt's keys and values, slices of the fused projection
        store("store_prompt", 16384, 4, 128, 64, "bf16", True),
        # one sequence read back in half precision
        fetch("fetch_sequence", 1037, 8, 64, 32, "fp16"),
        # a long context read back whole
        fetch("fetch_long", 131072, 4, 128, 64, "bf16"),
        # decoding one sequence after a prompt of about a thousand tokens
        attend("decode_one", 1, (1, 1), (1152, 1152), 4, 8, 128, 64, "bf16", True),
        # a decode step of 64 sequences of all lengths up to 4096
        attend("decode_batch", 64, (1, 1), (97, 4096), 4, 8, 128, 64, "bf16", True),
        # decoding one sequence over a long context
        attend("decode_long", 1, (1, 1), (131072, 131072), 4, 8, 128, 64, "bf16", False),
        # speculative verification: five rows of one sequence
        attend("verify", 1, (5, 5), (8191, 8191), 4, 8, 128, 16, "bf16", True),
        # odd group, small heads, half precision, odd pages, one sequence empty
        attend("decode_odd", 32, (1, 3), (5, 2003), 4, 5, 64, 48, "fp16", False, hole=True),
        # prompts fed in chunks of 64 rows at different depths, one sequence
        # shorter than its rows
        attend("chunk", 16, (37, 64), (70, 1149), 4, 8, 128, 64, "bf16", True, hole=True),
        # a whole prompt over its own freshly written cache
        attend("prompt", 1, (16384, 16384), (16384, 16384), 4, 8, 128, 64, "bf16", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page = rng.choice([16, 32, 48, 64, 128, 256])
    head_dim = rng.choice([64, 128, 128])
    op = rng.choice(["store", "fetch", "decode", "decode", "chunk"])
    if op == "store":
        kv_heads = rng.choice([1, 2, 4, 8])
        tokens = _log_int(rng, 1, 16384 * 4 * 128 // (max(kv_heads, 4) * head_dim))
        return {"op": "store", "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": page, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])
                if tokens <= 8192 else "bf16",
                "fused": rng.random() < 0.5, "padded": rng.choice([0, 0, tokens // 7])}
    if op == "fetch":
        kv_heads = rng.choice([1, 2, 4, 8])
        tokens = _log_int(rng, 1, 65536 * 4 // max(kv_heads, 4))
        return {"op": "fetch", "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": page, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    group = rng.choice([1, 2, 3, 5, 8, 16])
    kv_heads = rng.choice([1, 2, 4] if group == 1 else [1, 2, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "decode":
        seqs = _log_int(rng, 1, 64)
        ctx_hi = _log_int(rng, 1, 262144 * 4 // (max(kv_heads, 4) * seqs) // 2)
        ctx_lo = rng.randint(max(1, ctx_hi // 8), ctx_hi)
        rows = (1, 1) if rng.random() < 0.6 else (1, rng.randint(2, 8))
    else:
        seqs = _log_int(rng, 1, 16)
        rows_hi = _log_int(rng, 9, 4096 // seqs)
        rows = (rng.randint(max(1, rows_hi // 2), rows_hi), rows_hi)
        ctx_lo = rows_hi
        ctx_hi = rows_hi + _log_int(rng, 1, 8192)
    return {"op": "attend", "seqs": seqs, "rows_lo": rows[0], "rows_hi": rows[1],
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "kv_heads": kv_heads, "group": group,
            "head_dim": head_dim, "page": page, "dtype": dtype, "fused": rng.random() < 0.5,
            "hole": seqs > 2 and rng.random() < 0.5}


def _spread(lo, hi, n, phase):
    """n whole numbers spread evenly over [lo, hi], the same for every seed."""
    return [lo + int((hi - lo + 1) * (((i + phase) * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lengths(case):
    """Rows and cached tokens of each sequence."""
    n = case["seqs"]
    rows = _spread(case["rows_lo"], case["rows_hi"], n, 0.3)
    ctx = [max(c, r) for c, r in zip(_spread(case["ctx_lo"], case["ctx_hi"], n, 0.9), rows)]
    if case["hole"]:
        ctx[n // 2] = 0               # a sequence without any token: its rows see nothing
        ctx[n // 3] = (rows[n // 3] + 1) // 2  # fewer tokens than rows: the first rows see nothing
    return rows, ctx


# ---- inputs ----------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _keys_values(shape, g, dtype):
    """Keys with a few strong channels, as after a head's norm and rotation,
    and plain values; both as the projections' type."""
    strength = torch.exp(0.6 * torch.randn(shape[-1], generator=g, device="cuda"))
    k = torch.randn(shape, generator=g, device="cuda") * strength
    v = torch.randn(shape, generator=g, device="cuda") * 0.5
    return k.to(dtype), v.to(dtype)


def _pool(pages, case, g):
    """A pool whose tokens have all been written at some time, page by page."""
    H, D, page = case["kv_heads"], case["head_dim"], case["page"]
    data = torch.empty((pages, H, page // 16, 17 * D), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (H * page * D))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        k, v = _keys_values((n, H, page // 16, 16, D), g, torch.bfloat16)
        data[p:p + n] = _tiles(k, v)
    return data


def prepare(case, seed):
    g = _generator(seed)
    H, D, page = case["kv_heads"], case["head_dim"], case["page"]
    dtype = _DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] in ("store", "fetch"):
        T = case["tokens"]
        pages = -(-T // page) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        first = seed % page  # the sequence starts inside a page
        at = torch.arange(first, first + T, device="cuda")
        slots = order[at // page] * page + at % page
        if case["op"] == "store":
            if case["fused"]:  # keys and values are slices of one projection's rows
                rows = torch.randn((T, 10 * H, D), generator=g, device="cuda").to(dtype)
                k, v = rows[:, 8 * H:9 * H], rows[:, 9 * H:]
                kk, vv = _keys_values((T, H, D), g, dtype)
                k.copy_(kk)
                v.copy_(vv)
            else:
                k, v = _keys_values((T, H, D), g, dtype)
            if case["padded"]:
                slots[torch.randperm(T, generator=g, device="cuda")[:case["padded"]]] = -1
            state.update(k=k, v=v)
            pool = torch.zeros((pages, H, page // 16, 17 * D), dtype=torch.uint8, device="cuda")
        else:
            pool = _pool(pages, case, g)
        state.update(pool=pool, slots=slots, dtype=dtype)
    else:
        rows, ctx = _lengths(case)
        need = [-(-c // page) for c in ctx]
        width = max(max(need), 1)
        pages = sum(need) + 2
        pool = _pool(pages, case, g)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros((len(ctx), width), dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        T, Hq = sum(rows), H * case["group"]
        q = torch.randn((T, Hq + 2 * H if case["fused"] else Hq, D), generator=g, device="cuda")
        q = (2.0 * q).to(dtype)[:, :Hq]
        cu = [0]
        for r in rows:
            cu.append(cu[-1] + r)
        state.update(pool=pool, q=q, table=table, rows=rows, ctx=ctx, max_q=max(rows),
                     kv_lens=torch.tensor(ctx, dtype=torch.int32, device="cuda"),
                     cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    if own:
        from moe_fused_inference_b200 import kv4
        state["cache"] = kv4.KV4Cache.wrap(state["pool"])
        if case["op"] == "attend":
            state["workspace"] = kv4.attention_workspace(case["seqs"], case["kv_heads"] * case["group"],
                                                         state["cache"], max_q=state["max_q"])
    return state


# ---- the plain forms --------------------------------------------------------------
def _quantise(x):
    """x (..., D) -> 4-bit codes (..., nb, 32) and exponent codes (..., nb), uint8."""
    b = x.float().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    amax = b.abs().amax(-1)
    finite = torch.isfinite(amax)
    t = torch.clamp(torch.where(finite, amax, torch.ones_like(amax)) / 6.0, min=1e-30)
    m, ex = torch.frexp(t)                    # t = m * 2^ex, m in [.5, 1)
    e = torch.where(m > 0.5, ex, ex - 1)      # ceil(log2 t)
    y = torch.where(finite[..., None], torch.ldexp(b, -e[..., None]), torch.zeros_like(b))
    a = y.abs()
    code = torch.zeros_like(y, dtype=torch.uint8)
    for edge in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
        code += (a >= edge).to(torch.uint8)
    code += (y < 0).to(torch.uint8) * 8
    return code, torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def _pack_rows(code, pieces):
    """Codes (..., nb, 32) -> bytes (..., nb * 16), pieces of a block spread over the row."""
    nb = code.shape[-2]
    two = code[..., 0::2] | (code[..., 1::2] << 4)
    two = two.reshape(*code.shape[:-1], pieces, 16 // pieces)
    return two.transpose(-3, -2).reshape(*code.shape[:-2], nb * 16)


def _values(raw, scale, pieces):
    """Bytes (..., nb * 16) and exponent codes (..., nb) -> 32-bit values (..., D)."""
    nb = scale.shape[-1]
    b = raw.reshape(*raw.shape[:-1], pieces, nb, 16 // pieces).transpose(-3, -2)
    b = b.reshape(*raw.shape[:-1], nb, 16)
    code = torch.stack((b & 15, b >> 4), -1).reshape(*raw.shape[:-1], nb, 32)
    grid = torch.tensor(_GRID + tuple(-x for x in _GRID), device=raw.device)
    s = torch.where(scale == 255, float("nan"), torch.exp2(scale.float() - 127.0))
    return (grid[code.int()] * s[..., None]).reshape(*raw.shape[:-1], nb * 32)


def _tiles(k, v):
    """Keys and values (..., 16, D) -> tiles of bytes (..., 17 * D)."""
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    parts = (_pack_rows(kc, 4), _pack_rows(vc, 8), ks, vs)
    return torch.cat([p.flatten(-2) for p in parts], -1)


def _sections(pool):
    """Views of a pool's tiles: key rows, value rows, key codes, value codes."""
    D = pool.shape[-1] // 17
    ends = (0, 8 * D, 16 * D, 16 * D + D // 2, 17 * D)
    return [pool[..., a:b].unflatten(-1, (16, (b - a) // 16)) for a, b in zip(ends, ends[1:])]


def _places(pool, slots):
    """Page, tile and row of each slot."""
    page = pool.shape[2] * 16
    return slots // page, slots % page // 16, slots % 16


def _plain_store(state):
    pool, slots = state["pool"], state["slots"]
    live = slots >= 0
    p, t, r = _places(pool, slots[live])
    kr, vr, ksc, vsc = _sections(pool)
    (kc, ks), (vc, vs) = _quantise(state["k"][live]), _quantise(state["v"][live])
    for view, new in ((kr, _pack_rows(kc, 4)), (vr, _pack_rows(vc, 8)), (ksc, ks), (vsc, vs)):
        view[p, :, t, r] = new
    return _plain_fetch(state)


def _plain_fetch(state):
    pool, slots = state["pool"], state["slots"]
    live = (slots >= 0)[:, None, None]
    p, t, r = _places(pool, slots.clamp(min=0))
    kr, vr, ksc, vsc = (s[p, :, t, r] for s in _sections(pool))
    return [torch.where(live, _values(raw, sc, n), 0.0).to(state["dtype"])
            for raw, sc, n in ((kr, ksc, 4), (vr, vsc, 8))]


def _plain_attend(state):
    q, pool, table = state["q"], state["pool"], state["table"]
    G, H, D = state["case"]["group"], state["case"]["kv_heads"], state["case"]["head_dim"]
    page = pool.shape[2] * 16
    out = torch.zeros((q.shape[0], q.shape[1], D), dtype=q.dtype, device=q.device)
    sections = _sections(pool)
    at = 0
    for i, (R, L) in enumerate(zip(state["rows"], state["ctx"])):
        first, at = at, at + R
        if R == 0 or L == 0:
            continue
        ids = table[i, :-(-L // page)].long()
        kr, vr, ksc, vsc = (s[ids].transpose(0, 1).flatten(1, 3)[:, :L] for s in sections)
        k, v = _values(kr, ksc, 4), _values(vr, vsc, 8)          # (H, L, D)
        step = max(1, (1 << 28) // (H * G * L))
        for r0 in range(0, R, step):
            n = min(step, R - r0)
            see = min(L, max(0, L - R + r0 + n))                 # tokens the last row sees
            if see == 0:
                continue
            qs = q[first + r0:first + r0 + n].float().reshape(n, H, G, D)
            qs = qs.permute(1, 2, 0, 3).reshape(H, G * n, D)
            s = torch.matmul(qs, k[:, :see].transpose(1, 2)) / math.sqrt(D)
            s = s.reshape(H, G, n, see)
            last = torch.arange(L - R + r0, L - R + r0 + n, device=q.device)
            dead = torch.arange(see, device=q.device) > last[:, None]
            s = torch.where(dead, -math.inf, s)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            norm = p.sum(-1, keepdim=True)
            o = torch.matmul(p.reshape(H, G * n, see), v[:, :see]).reshape(H, G, n, D)
            o = torch.where(norm > 0, o / torch.where(norm > 0, norm, 1.0), 0.0)
            o = torch.where(norm.isnan(), math.nan, o)
            out[first + r0:first + r0 + n] = o.permute(2, 0, 1, 3).reshape(n, H * G, D).to(q.dtype)
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"store": _plain_store, "fetch": _plain_fetch, "attend": _plain_attend}[op](state)
    from moe_fused_inference_b200 import kv4
    cache = state["cache"]
    if op == "store":
        kv4.kv4_write(cache, state["k"], state["v"], state["slots"])
        return list(kv4.kv4_read(cache, state["slots"], dtype=state["dtype"]))
    if op == "fetch":
        return list(kv4.kv4_read(cache, state["slots"], dtype=state["dtype"]))
    return kv4.kv4_attention(state["q"], cache, state["table"], state["kv_lens"],
                             cu_q=state["cu_q"], max_q=state["max_q"],
                             workspace=state["workspace"])


# ---- what a pass cannot do without --------------------------------------------------
def work(case):
    H, D = case["kv_heads"], case["head_dim"]
    held = 2 * (D // 2 + D // 32)                 # bytes of one token's key and value, one head
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "store":   # read k and v, write the cache, read it, write the values
        T, live = case["tokens"], case["tokens"] - case["padded"]
        return {"bytes": T * (H * 2 * D * size + 8) + live * H * (2 * held + 2 * D * size)
                + case["padded"] * H * 2 * D * size, "flops": 0}
    if case["op"] == "fetch":
        return {"bytes": case["tokens"] * (H * (held + 2 * D * size) + 8), "flops": 0}
    rows, ctx = _lengths(case)
    Hq = H * case["group"]
    seen = 0
    for R, L in zip(rows, ctx):  # tokens seen, summed over the rows
        full = max(0, L - R)
        n = min(R, L)            # rows that see something
        seen += n * full + (n * (n + 1) // 2)
    return {"bytes": sum(ctx) * H * held + 2 * sum(rows) * Hq * D * size
            + 4 * sum(-(-c // case["page"]) for c in ctx) + 8 * len(ctx),
            "flops": 4 * seen * Hq * D}


# ---- the definition in 64 bits --------------------------------------------------------
def _exact_block(x):
    """Values (..., 32) in 64 bits -> what their block holds of them."""
    top = x.abs().max(dim=-1, keepdim=True).values
    e = torch.full_like(top, -99.0)
    for b in (128, 64, 32, 16, 8, 4, 2, 1):       # smallest e with 6 * 2^e >= top
        e = torch.where(6.0 * torch.exp2(e + (b - 1)) < top, e + b, e)
    scale = torch.exp2(e)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    best = torch.zeros_like(x)
    gap = torch.full_like(x, math.inf)
    for m in grid:                                # the later, larger one wins a tie
        d = (x.abs() / scale - m).abs()
        best = torch.where(d <= gap, m, best)
        gap = torch.minimum(d, gap)
    return torch.sign(x) * best * scale


def _exact_heads(tiles, D):
    """Tiles of bytes (..., 17 * D) -> keys and values (..., 16, D) in 64 bits,
    each element looked up at the byte and the half that the layout names."""
    el = torch.arange(D, device=tiles.device)
    blk, i, nb = el // 32, el % 32, D // 32
    row = torch.arange(16, device=tiles.device)[:, None]
    table = torch.tensor([s * m for s in (1.0, -1.0) for m in _GRID], dtype=torch.float64,
                         device=tiles.device)
    out = []
    for base, codes, at in ((0, 16 * D, ((i // 8) * nb + blk) * 4 + (i % 8) // 2),
                            (8 * D, 16 * D + D // 2, ((i // 4) * nb + blk) * 2 + (i % 4) // 2)):
        byte = tiles[..., base + row * (D // 2) + at].long()
        nib = torch.where(i % 2 == 0, byte % 16, byte // 16)
        power = tiles[..., codes + row * nb + blk].double() - 127.0
        out.append(table[nib] * torch.exp2(power))
    return out


def exact(case, seed):
    state = prepare(case, seed)
    D, H = case["head_dim"], case["kv_heads"]
    if case["op"] == "store":
        live = (state["slots"] >= 0)[:, None, None]
        outs = []
        for x in (state["k"], state["v"]):
            x = x.double()
            outs.append(_exact_block(x.reshape(*x.shape[:-1], -1, 32)).reshape(x.shape) * live)
        return outs
    pool = state["pool"]
    tiles_per_page = pool.shape[2]
    flat = pool.transpose(1, 2).reshape(-1, H, 17 * D)  # tile of the pool, head, bytes
    if case["op"] == "fetch":
        outs = ([], [])
        for part in state["slots"].split(8192):
            tile, row = part // 16, part % 16
            for o, x in zip(outs, _exact_heads(flat[tile], D)):
                o.append(x[torch.arange(len(part), device=x.device), :, row])
        return [torch.cat(o) for o in outs]
    out = torch.zeros((state["q"].shape[0], H * case["group"], D), dtype=torch.float64, device="cuda")
    start = 0
    for i, (R, L) in enumerate(zip(state["rows"], state["ctx"])):
        ids = state["table"][i, :(L + case["page"] - 1) // case["page"]].long()
        tiles = (ids[:, None] * tiles_per_page
                 + torch.arange(tiles_per_page, device="cuda")).reshape(-1)[:(L + 15) // 16]
        for h in range(H if L else 0):
            k, v = (x.reshape(-1, D)[:L] for x in _exact_heads(flat[tiles, h], D))
            for j in range(h * case["group"], (h + 1) * case["group"]):
                for a in range(max(0, R - L), R, 4096):
                    b = min(R, a + 4096)
                    sees = L - R + b                     # tokens the part's last row sees
                    w = state["q"][start + a:start + b, j].double() @ k[:sees].T * D ** -0.5
                    keep = torch.ones_like(w, dtype=torch.bool).tril(L - R + a)
                    w = torch.softmax(w.masked_fill(~keep, -math.inf), dim=1)
                    out[start + a:start + b, j] = w @ v[:sees]
        start += R
    return out
