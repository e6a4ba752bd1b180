"""The serving-side attention operators, as cases that can be timed and compared.

Four operators that a decoding step runs in this order:

  tables     block tables, slots and positions of a step's new tokens, from the requests' lengths
  append     rotary positions on q and k, and k and v written into the paged key-value cache
  attention  one new token per request against its pages, split over the length and joined
  rope       the same rotary positions on their own, forward and as the gradient (before prefill
             attention, and in its backward pass)

``run`` computes them with elementary torch operations (``own`` false) or with this package's
kernels (``own`` true), from the state that ``prepare`` made.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
          "e4m3": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # a small serving batch, one token each: the call whose latency counts
        _tables("tables decode 8", decode=8, prefill=0, release=0, chunk=1, lo=20, hi=900, block=16),
        # continuous batching: most requests decode, some bring a chunk of their prompt, some are done
        _tables("tables mixed 256", decode=200, prefill=40, release=16, chunk=257, lo=1, hi=5000,
                block=16),
        # offline scoring: many long prompts at once
        _tables("tables prompts 64", decode=0, prefill=64, release=64, chunk=2040, lo=1, hi=3,
                block=32),
        # queries of a video model before attention: time, height, width; heads before positions
        _rope("rope video bf16", dtype="bf16", batch=4, seq=4096, heads=32, dim=128, rot=128,
              axes=3, interleaved=False, inverse=False, heads_first=True, far=4096),
        # the gradient in 32 bits, image patches (height, width) in adjacent pairs, odd sizes
        _rope("rope image gradient f32", dtype="f32", batch=3, seq=1013, heads=12, dim=80, rot=80,
              axes=2, interleaved=True, inverse=True, heads_first=False, far=200),
        # one token of each of 64 requests, q, k and v of one projection
        _append("append decode 64", dtype="bf16", cache="bf16", tokens=64, heads=32, kv_heads=8,
                dim=128, rot=128, axes=1, interleaved=False, block=16, far=100000, skip=0),
        # a prefill chunk into a cache of 8 bits, three axes
        _append("append prefill e4m3", dtype="bf16", cache="e4m3", tokens=8192, heads=32,
                kv_heads=8, dim=128, rot=128, axes=3, interleaved=False, block=64, far=30000,
                skip=0),
        # an odd chunk, a quarter of each head rotated, some rows padding
        _append("append padded f16", dtype="f16", cache="f16", tokens=1021, heads=16, kv_heads=16,
                dim=64, rot=32, axes=1, interleaved=True, block=16, far=2000, skip=29),
        # one request, a short context
        _attention("attention one short", dtype="bf16", cache="bf16", requests=1, heads=32,
                   kv_heads=8, dim=128, lo=700, hi=700, empty=0, block=16, window=0,
                   heads_first=False),
        # a batch whose lengths spread over three decades, some slots of it empty
        _attention("attention ragged 128", dtype="f16", cache="f16", requests=128, heads=16,
                   kv_heads=4, dim=64, lo=8, hi=16001, empty=5, block=16, window=0,
                   heads_first=True),
        # few requests with long contexts, a cache of 8 bits
        _attention("attention long e4m3", dtype="bf16", cache="e4m3", requests=3, heads=64,
                   kv_heads=8, dim=128, lo=90001, hi=131072, empty=0, block=64, window=0,
                   heads_first=False),
        # a full batch at steady state: the largest
        _attention("attention batch 64", dtype="bf16", cache="bf16", requests=64, heads=32,
                   kv_heads=8, dim=128, lo=7900, hi=8190, empty=0, block=16, window=0,
                   heads_first=False),
    ]


def _tables(name, **c):
    return {"name": name, "op": "tables", **c}


def _rope(name, **c):
    return {"name": name, "op": "rope", **c}


def _append(name, **c):
    return {"name": name, "op": "append", **c}


def _attention(name, **c):
    return {"name": name, "op": "attention", **c}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "rope", "append", "attention", "attention"])
    if op == "tables":
        lo = _log(rng, 1, 1000)
        c = {"op": op, "decode": _log(rng, 1, 600) if rng.random() < 0.8 else 0,
             "prefill": _log(rng, 1, 64) if rng.random() < 0.6 else 0,
             "release": _log(rng, 1, 64) if rng.random() < 0.5 else 0,
             "chunk": _log(rng, 2, 2040), "lo": lo, "hi": _log(rng, lo, 6000),
             "block": rng.choice([8, 16, 32, 64, 24, 1])}
        c["decode"] += 1 if c["decode"] + c["prefill"] == 0 else 0
        return c
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads = rng.choice([1, 2, 5, 8, 12, 24, 32])
        batch = _log(rng, 1, 8)
        most = min(16384, (1 << 26) // (dim * heads * batch))
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "batch": batch,
                "seq": _log(rng, 1, most), "heads": heads, "dim": dim,
                "rot": rng.choice([dim, dim // 2 // 16 * 16]), "axes": rng.choice([1, 2, 3, 4]),
                "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.5,
                "heads_first": rng.random() < 0.5, "far": _log(rng, 10, 1000000)}
    dtype = rng.choice(["bf16", "f16"])
    cache = rng.choice([dtype, dtype, "e4m3"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    dim = rng.choice([64, 128, 128, 256])
    block = rng.choice([8, 16, 32, 64, 24, 1])
    if op == "append":
        tokens = _log(rng, 1, min(16384, (1 << 25) // ((heads + 2 * kv_heads) * dim)))
        return {"op": op, "dtype": dtype, "cache": cache, "tokens": tokens, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rot": rng.choice([dim, dim // 2]),
                "axes": rng.choice([1, 1, 3]), "interleaved": rng.random() < 0.3, "block": block,
                "far": _log(rng, 10, 1000000), "skip": tokens // 20}
    requests = _log(rng, 1, 256)
    most = min(131072, (1 << 28) // (requests * kv_heads * dim))
    hi = _log(rng, 1, max(1, most))
    return {"op": op, "dtype": dtype, "cache": cache, "requests": requests, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "lo": _log(rng, 1, hi), "hi": hi,
            "empty": requests // 10, "block": block,
            "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
            "heads_first": rng.random() < 0.5}


def _spread(n, lo, hi):
    """n lengths spread evenly over the logarithm of lo..hi (the seed only orders them)."""
    if n <= 1:
        return [hi] * n
    return [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _request_lengths(c):
    """(length, new tokens) of the requests of a tables case; -1 new tokens release a request."""
    d, p, r = c["decode"], c["prefill"], c["release"]
    rows = [(n, 1) for n in _spread(d, c["lo"], c["hi"])]
    rows += [(n, max(1, c["chunk"] - i)) for i, n in enumerate(_spread(p, c["lo"], c["hi"]))]
    rows += [(n, -1) for n in _spread(r, c["lo"], c["hi"])]
    return rows


def _cache_lengths(c):
    n = c["requests"] - c["empty"]
    return _spread(n, c["lo"], c["hi"]) + [0] * c["empty"]


def _blocks(n, block):
    return -(-n // block)


# -------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "tables":
        rows = _request_lengths(c)
        tokens = sum(max(n, 0) for _, n in rows)
        fresh = sum(_blocks(m + n, c["block"]) - _blocks(m, c["block"]) for m, n in rows if n > 0)
        freed = sum(_blocks(m, c["block"]) for m, n in rows if n < 0)
        # lengths, counts, status and sums; slot, position and request of each token; the free
        # blocks read and written into the table; the freed ones read and pushed
        return {"bytes": 20 * len(rows) + 12 * tokens + 8 * fresh + 8 * freed, "flops": 0}
    if c["op"] == "rope":
        n = c["batch"] * c["seq"] * c["heads"]
        angles = c["batch"] * c["seq"] * c["axes"] * 4
        return {"bytes": 2 * n * c["dim"] * SIZE[c["dtype"]] + angles, "flops": 3 * n * c["rot"]}
    if c["op"] == "append":
        t, h, g, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        live = t - c["skip"]
        e, s = SIZE[c["dtype"]], SIZE[c["cache"]]
        return {"bytes": (2 * t * h + 2 * live * g) * d * e + 2 * live * g * d * s
                + t * (c["axes"] + 1) * 4,
                "flops": 3 * (t * h + live * g) * c["rot"]}
    keys = sum(min(n, c["window"]) if c["window"] else n for n in _cache_lengths(c))
    pages = sum(_blocks(n, c["block"]) for n in _cache_lengths(c))
    return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] * SIZE[c["cache"]] + 4 * pages
            + 2 * c["requests"] * c["heads"] * c["dim"] * SIZE[c["dtype"]],
            "flops": 4 * keys * c["heads"] * c["dim"]}


# ----------------------------------------------------------------------------- prepare
def _randn(g, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.bfloat16
                    if dtype == "e4m3" else DTYPES[dtype])
    if dtype == "e4m3":
        return (x * 16).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return x if scale == 1.0 else x.mul_(scale)


def _order(g, n):
    return torch.randperm(n, generator=g, device=DEVICE)


def _frequencies(rot):
    i = torch.arange(rot // 2, dtype=torch.float64)
    return 10000.0 ** (-2.0 * i / rot)


def _axes(rot, axes):
    """Which axis each frequency follows: neighbouring runs of frequencies, as for video."""
    return (torch.arange(rot // 2) * axes // (rot // 2)).to(torch.int32)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "tables":
        rows = _request_lengths(c)
        both = torch.tensor(rows, dtype=torch.int32, device=DEVICE)[_order(g, len(rows))]
        s["lens"], s["new"] = both[:, 0].contiguous(), both[:, 1].contiguous()
        held = [_blocks(m, c["block"]) for m, _ in rows]
        s["max_blocks"] = max(_blocks(m + max(n, 0), c["block"]) for m, n in rows)
        fresh = sum(_blocks(m + n, c["block"]) - _blocks(m, c["block"]) for m, n in rows if n > 0)
        total = sum(held) + fresh + 3
        ids = _order(g, total).to(torch.int32)
        mine = _blocks_of(s["lens"], c["block"]).long()
        first = mine.cumsum(0) - mine
        j = torch.arange(s["max_blocks"], device=DEVICE)
        at = (first[:, None] + j).clamp(max=total - 1)
        s["table"] = torch.where(j < mine[:, None], ids[at], -1).contiguous()
        # the stack of free blocks: the first ones free, room for the rest above them
        s["free"] = torch.cat([ids[sum(held):], ids.new_full((sum(held),), -1)])
        s["free_count"] = torch.tensor([total - sum(held)], dtype=torch.int32, device=DEVICE)
        s["max_tokens"] = sum(max(n, 0) for _, n in rows)
        return s
    if c["op"] == "rope":
        b, n, h, d = c["batch"], c["seq"], c["heads"], c["dim"]
        shape = (b, h, n, d) if c["heads_first"] else (b, n, h, d)
        x = _randn(g, shape, c["dtype"])
        s["x"] = x.transpose(1, 2) if c["heads_first"] else x
        s["pos"] = torch.randint(0, c["far"], (c["axes"], b, n), generator=g, device=DEVICE,
                                 dtype=torch.int32)
        s["freq"], s["axis"] = _frequencies(c["rot"]), _axes(c["rot"], c["axes"])
        return s
    if c["op"] == "append":
        t, h, kv, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        qkv = _randn(g, (t, (h + 2 * kv) * d), c["dtype"])
        s["q"] = qkv[:, :h * d].view(t, h, d)
        s["k"] = qkv[:, h * d:(h + kv) * d].view(t, kv, d)
        s["v"] = qkv[:, (h + kv) * d:].view(t, kv, d)
        s["pos"] = torch.randint(0, c["far"], (c["axes"], t), generator=g, device=DEVICE,
                                 dtype=torch.int32)
        nb = _blocks(t, c["block"]) + 2
        slots = _order(g, nb * c["block"])[:t].to(torch.int32)
        if c["skip"]:
            slots[-c["skip"]:] = -1
        s["slots"] = slots
        for name in ("kc", "vc"):
            s[name] = _randn(g, (nb, c["block"], kv, d), c["cache"])
        s["freq"], s["axis"] = _frequencies(c["rot"]), _axes(c["rot"], c["axes"])
        s["k_scale"], s["v_scale"] = (0.03, 0.05) if c["cache"] == "e4m3" else (1.0, 1.0)
        return s
    lens = _cache_lengths(c)
    kv, d, block = c["kv_heads"], c["dim"], c["block"]
    s["longest"] = max(lens)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)[_order(g, len(lens))]
    mine = _blocks_of(s["lens"], block).long()
    total = sum(_blocks(n, block) for n in lens) + 1
    ids = _order(g, total).to(torch.int32)
    j = torch.arange(max(1, _blocks(s["longest"], block)), device=DEVICE)
    at = ((mine.cumsum(0) - mine)[:, None] + j).clamp(max=total - 1)
    s["table"] = torch.where(j < mine[:, None], ids[at], -1).contiguous()
    shape = (total, kv, block, d) if c["heads_first"] else (total, block, kv, d)
    for name in ("kc", "vc"):
        x = _randn(g, shape, c["cache"])
        s[name] = x.transpose(1, 2) if c["heads_first"] else x
    s["q"] = _randn(g, (c["requests"], c["heads"], d), c["dtype"], 2.0)
    s["k_scale"], s["v_scale"] = (0.07, 0.05) if c["cache"] == "e4m3" else (1.0, 1.0)
    s["scale"] = d ** -0.5
    return s


def _blocks_of(lens, block):
    return (lens + (block - 1)) // block


# --------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "rope": _own_rope, "append": _own_append,
                "attention": _own_attention}[op](state)
    return {"tables": _plain_tables, "rope": _plain_rope, "append": _plain_append,
            "attention": _plain_attention}[op](state)


def _own_tables(s):
    import remora_b200 as rb
    r = rb.kv_block_table(s["lens"], s["new"], s["table"], s["free"], s["free_count"],
                          block_size=s["case"]["block"], max_tokens=s["max_tokens"])
    return {"lens": r.lens, "free_count": r.free_count, "cu": r.cu_tokens, "slots": r.slots,
            "positions": r.positions, "requests": r.requests, "status": r.status,
            "table": s["table"], "free": s["free"]}


def _own_rope(s):
    import remora_b200 as rb
    c = s["case"]
    return rb.rope(s["x"], s["pos"], s["freq"], axis_of=s["axis"], interleaved=c["interleaved"],
                   inverse=c["inverse"])


def _own_append(s):
    import remora_b200 as rb
    q = rb.rope_kv_append(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["freq"], s["kc"],
                          s["vc"], axis_of=s["axis"], interleaved=s["case"]["interleaved"],
                          k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _own_attention(s):
    import remora_b200 as rb
    c = s["case"]
    lse = torch.empty((c["requests"], c["heads"]), dtype=torch.float32, device=s["q"].device)
    out = rb.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], scale=s["scale"],
                             window=c["window"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                             lse=lse)
    return {"out": out, "lse": lse}


def _plain_tables(s):
    block, most = s["case"]["block"], s["max_tokens"]
    lens, new, table, free = s["lens"].long(), s["new"].long(), s["table"], s["free"]
    n_free = s["free_count"].long()
    dev = lens.device
    gone = new == -1
    n = new.clamp(min=0)
    ends = n.cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends])
    held = _blocks_of(lens, block)
    # blocks of released requests go on the stack in request order
    back = torch.where(gone, held, 0)
    back_ends = back.cumsum(0)
    j = torch.arange(free.numel(), device=dev)
    who = torch.searchsorted(back_ends, j - n_free, right=True).clamp(max=lens.numel() - 1)
    which = (j - n_free - (back_ends - back)[who]).clamp(0, table.shape[1] - 1)
    pushed = (j >= n_free) & (j < n_free + back_ends[-1])
    free.copy_(torch.where(pushed, table[who, which], free))
    have = n_free + back_ends[-1]
    # requests take what they need from the top of the stack, in request order
    fits = (lens + n <= table.shape[1] * block) & (ends <= most) & ~gone
    need = torch.where(fits, _blocks_of(lens + n, block) - held, 0)
    need_ends = need.cumsum(0)
    granted = fits & ((need == 0) | (need_ends <= have))
    taken = torch.where(granted & (need > 0), need_ends, 0).max()
    status = torch.where(granted | gone, 0, torch.where(fits, 1, 2))
    # each token
    t = torch.arange(most, device=dev)
    r = torch.searchsorted(ends, t, right=True)
    real = r < lens.numel()
    r = r.clamp(max=lens.numel() - 1)
    p = lens[r] + t - cu[r]
    ok = real & granted[r]
    page = torch.where(ok, p // block, 0)
    fresh = page - held[r]
    spot = (have - 1 - ((need_ends - need)[r] + fresh)).clamp(0, free.numel() - 1)
    ids = torch.where(fresh >= 0, free[spot], table[r, page.clamp(max=table.shape[1] - 1)])
    first = ok & (fresh >= 0) & (p % block == 0)
    # a token that opens no block writes to a cell past the table
    flat = torch.cat([table.reshape(-1), table.new_zeros(1)])
    flat[torch.where(first, r * table.shape[1] + page, table.numel())] = ids
    table.copy_(flat[:-1].view_as(table))
    i32 = torch.int32
    return {"lens": torch.where(gone, 0, torch.where(granted, lens + n, lens)).to(i32),
            "free_count": (have - taken).to(i32), "cu": cu.to(i32),
            "slots": torch.where(ok, ids * block + p % block, -1).to(i32),
            "positions": torch.where(ok, p, 0).to(i32),
            "requests": torch.where(real, r, -1).to(i32), "status": status.to(i32),
            "table": table, "free": free}


def _angles(pos, freq, axis):
    """cos and sin of each token's angles in 32 bits, the angles in 64: [..., rot / 2]."""
    a = pos[axis.long().to(pos.device)].double().movedim(0, -1) * freq.to(pos.device)
    return a.cos().float(), a.sin().float()


def _rotated(x, cos, sin, interleaved):
    """x [..., heads, dim] in 32 bits, its first 2 * cos.shape[-1] elements rotated in pairs."""
    half = cos.shape[-1]
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = turn[..., :half], turn[..., half:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, rest], -1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = _angles(s["pos"], s["freq"], s["axis"])
    y = _rotated(s["x"].float(), cos, -sin if c["inverse"] else sin, c["interleaved"])
    return y.to(s["x"].dtype)


def _stored(x, scale, dtype):
    if dtype == torch.float8_e4m3fn:
        return (x / scale).clamp(-448, 448).to(dtype)
    return x.to(dtype)


def _put(cache, slots, rows):
    """Rows at their slots; a row without one goes to a cell past the cache."""
    n = cache.shape[0] * cache.shape[1]
    flat = cache.view(torch.uint8).view(n, -1)
    more = torch.cat([flat, flat.new_zeros(1, flat.shape[1])])
    more[torch.where(slots >= 0, slots, n).long()] = rows.contiguous().view(torch.uint8).view(
        rows.shape[0], -1)
    flat.copy_(more[:-1])


def _plain_append(s):
    inter = s["case"]["interleaved"]
    cos, sin = _angles(s["pos"], s["freq"], s["axis"])
    q = _rotated(s["q"].float(), cos, sin, inter).to(s["q"].dtype)
    k = _rotated(s["k"].float(), cos, sin, inter)
    _put(s["kc"], s["slots"], _stored(k, s["k_scale"], s["kc"].dtype))
    _put(s["vc"], s["slots"], _stored(s["v"].float(), s["v_scale"], s["vc"].dtype))
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _pages(cache, page, off, scale):
    """The rows of the cache in 32 bits: [requests, length, kv heads, dim]."""
    if cache.dtype == torch.float8_e4m3fn:
        rows = cache.view(torch.uint8)[page, off].view(torch.float8_e4m3fn)
        return rows.float() * scale
    return cache[page, off].float()


def _plain_attention(s):
    c = s["case"]
    r, h, d = s["q"].shape
    kv, block = c["kv_heads"], c["block"]
    pos = torch.arange(s["longest"], device=s["q"].device)
    page = s["table"][:, pos // block].long().clamp(min=0)
    keys = _pages(s["kc"], page, pos % block, s["k_scale"]).transpose(1, 2)
    q = s["q"].float().view(r, kv, h // kv, d)
    score = torch.matmul(q, keys.transpose(2, 3)) * s["scale"]
    del keys
    lens = s["lens"].long()[:, None]
    seen = pos < lens
    if c["window"]:
        seen = seen & (pos >= lens - c["window"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    values = _pages(s["vc"], page, pos % block, s["v_scale"]).transpose(1, 2)
    out = torch.matmul(p / torch.where(total == 0, 1.0, total), values)
    lse = (top + torch.log(total)).view(r, h)
    return {"out": out.view(r, h, d).to(s["q"].dtype), "lse": lse}


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    """What run() returns, computed request by request or token by token in 64 bits."""
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "tables":
        return None  # whole numbers
    if c["op"] == "rope":
        y = _turned(s["x"].double(), s["pos"], s, c["interleaved"], -1.0 if c["inverse"] else 1.0)
        return y
    if c["op"] == "append":
        q = _turned(s["q"].double(), s["pos"], s, c["interleaved"], 1.0)
        k = _turned(s["k"].double(), s["pos"], s, c["interleaved"], 1.0) / s["k_scale"]
        v = s["v"].double() / s["v_scale"]
        live = (s["slots"] >= 0).nonzero()[:, 0]
        at = s["slots"][live].long()
        found = {"q": q}
        for name, cache, rows in (("k_cache", s["kc"], k), ("v_cache", s["vc"], v)):
            flat = cache.double().flatten(0, 1)
            if c["cache"] == "e4m3":
                rows = rows.clamp(-448, 448)
            flat[at] = rows[live]
            found[name] = flat.view(cache.shape)
        return found
    r, h, d = s["q"].shape
    kv, block = c["kv_heads"], c["block"]
    out = torch.zeros((r, h, d), dtype=torch.float64, device=DEVICE)
    lse = torch.full((r, h), -math.inf, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][i, :_blocks(n, block)].long()
        start = max(0, n - c["window"]) if c["window"] else 0
        for g in range(kv):
            k = s["kc"].view(torch.uint8)[pages][:, :, g] if c["cache"] == "e4m3" else \
                s["kc"][pages][:, :, g]
            v = s["vc"].view(torch.uint8)[pages][:, :, g] if c["cache"] == "e4m3" else \
                s["vc"][pages][:, :, g]
            if c["cache"] == "e4m3":
                k, v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
            k = k.reshape(-1, d)[start:n].double() * s["k_scale"]
            v = v.reshape(-1, d)[start:n].double() * s["v_scale"]
            rows = slice(g * (h // kv), (g + 1) * (h // kv))
            score = s["q"][i, rows].double() @ k.t() * s["scale"]
            lse[i, rows] = torch.logsumexp(score, -1)
            out[i, rows] = torch.softmax(score, -1) @ v
    return {"out": out, "lse": lse}


def _turned(x, pos, s, interleaved, sign):
    """Each pair as a complex number, turned by its angle."""
    rot, dim = 2 * s["freq"].numel(), x.shape[-1]
    angle = torch.stack([pos[a].double() * f for a, f in zip(s["axis"].tolist(),
                                                             s["freq"].tolist())], -1)
    turn = torch.polar(torch.ones_like(angle), sign * angle).unsqueeze(-2)
    low = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    high = low + 1 if interleaved else low + rot // 2
    z = torch.complex(x[..., low], x[..., high]) * turn
    y = x.clone()
    y[..., low], y[..., high] = z.real, z.imag
    return y if rot <= dim else None
