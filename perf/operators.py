"""The operators between a decoder's q|k|v linear and its o linear, over a key/value cache held in 4 bits: their plain
forms in elementary torch operations, the calls of this package that do the same, and the cases they are measured on.

``plan``       page tables, slot maps and positions of one step, built on the GPU from the requests' lengths
``norm_rope``  per-head norms of q and k with the position rotation
``store``      the same, with k and v quantised into the cache; the stored rows are read back as the values they stand for
``attention``  attention of the new rows over the cached ones

A page of the cache holds ``page`` tokens; per page and kv head it is a run of blocks of 16 tokens, 18 * D bytes each:
K codes ``[16 tokens][D/2]`` (two E2M1 per byte, even dimension in the low nibble), V codes ``[2][8][4][2][D/16]`` (token
8p + 2t + j, bytes of dimensions g*D/8 .., at ``[p][g][t][j]``), K scales ``[8][4][2][D/64]`` (E4M3; token 8h + r, group
t*D/64 + i at ``[r][t][h][i]``), V scales ``[D/16][4][2][2]`` (group, t, p, j). A value is code * scale / divisor."""
import math
import random

import torch

own = False

DEV = "cuda"
KDIV, VDIV, EPS = 16.0, 16.0, 1e-6
_backend = None


# ---- the cases -------------------------------------------------------------------------------------------------------

def _plan(name, requests, new, context, page, spare):
    return {"name": name, "op": "plan", "requests": requests, "new_min": new[0], "new_max": new[1], "context_min": context[0],
            "context_max": context[1], "page": page, "spare_rows": spare}


def _rope(name, tokens, dtype, heads, kv_heads, head_dim, rot, interleaved):
    return {"name": name, "op": "norm_rope", "tokens": tokens, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rot": rot, "interleaved": interleaved}


def _store(name, tokens, dtype, heads, kv_heads, head_dim, page):
    return {"name": name, "op": "store", "tokens": tokens, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rot": head_dim, "interleaved": False, "page": page}


def _attention(name, requests, new, context, heads, kv_heads, head_dim, page, causal=True, window=0, spare=0):
    return {"name": name, "op": "attention", "requests": requests, "new_min": new[0], "new_max": new[1], "context_min": context[0],
            "context_max": context[1], "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "causal": causal,
            "window": window, "spare_rows": spare}


def listed():
    return [
        # one decode step of a server's running batch: a page is taken now and then
        _plan("plan 64 decoding", 64, (1, 1), (17, 8000), 64, 0),
        # a large ragged admission step, padded to a fixed token count as a captured graph needs it
        _plan("plan 1000 ragged", 1000, (0, 70), (0, 4000), 16, 333),
        # decode batch behind the bf16 twins of the q|k|v linear (the stack's 64 / 8 heads of 128)
        _rope("norm+rope 32 decode bf16", 32, "bf16", 64, 8, 128, 128, False),
        # a prefill step in the f32 buffers, half of each head rotated, neighbouring pairs
        _rope("norm+rope 1999 f32", 1999, "f32", 32, 4, 128, 64, True),
        # decode batch and prefill step with the write into the cache
        _store("store 48 decode", 48, "bf16", 64, 8, 128, 64),
        _store("store 2048 prefill", 2048, "bf16", 64, 8, 128, 64),
        # one user, one token, a short chat: latency
        _attention("decode 1 x 1000", 1, (1, 1), (1000, 1000), 64, 8, 128, 64),
        # a full decode batch with ragged contexts
        _attention("decode 64 x 8k ragged", 64, (1, 1), (4000, 8200), 64, 8, 128, 64),
        # few very long contexts: the sequence has to be split
        _attention("decode 3 x 130k", 3, (1, 1), (9001, 130001), 64, 8, 128, 128),
        # a drafter's tokens verified in one step, smaller heads, sliding window, ungrouped by eight
        _attention("verify 24 x 3 window", 24, (1, 3), (50, 6000), 28, 4, 64, 16, True, 1024, 5),
        # a chunk of a long prompt behind what is cached of it
        _attention("chunk 2048 of 8192", 1, (2048, 2048), (8192, 8192), 64, 8, 128, 64),
        # chunked prefill of several prompts next to decoding requests
        _attention("mixed 12 chunks", 12, (1, 300), (300, 9000), 64, 8, 128, 32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


_HEADS = [(64, 8), (32, 4), (16, 2), (8, 1), (8, 8), (28, 4), (16, 1), (10, 2)]


def draw(rng):
    op = rng.choice(["plan", "norm_rope", "store", "attention", "attention", "attention"])
    heads, kv_heads = rng.choice(_HEADS)
    head_dim, page = rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "plan":
        c = _plan("", _log(rng, 1, 1200), (0, _log(rng, 1, 60)), (0, _log(rng, 10, 9000)), page, _log(rng, 1, 400))
    elif op == "norm_rope":
        c = _rope("", _log(rng, 1, 2000), dtype, heads, kv_heads, head_dim, rng.choice([head_dim, head_dim, head_dim // 2]), rng.random() < 0.3)
    elif op == "store":
        c = _store("", _log(rng, 1, 2000), dtype, heads, kv_heads, head_dim, page)
    elif rng.random() < 0.6:   # decode and verify widths
        b = _log(rng, 1, 64)
        most = max(64, min(100000, 200000 // b))
        c = _attention("", b, (1, rng.choice([1, 1, 1, 2, 5])), (1, _log(rng, 20, most)), heads, kv_heads, head_dim, page, True,
                       rng.choice([0, 0, 0, 500]), _log(rng, 1, 9) - 1)
    else:
        b = _log(rng, 1, 8)
        new = _log(rng, 17, 1500 // b)
        c = _attention("", b, (1, new), (new, new + _log(rng, 1, 6000 // b)), heads, kv_heads, head_dim, page, rng.random() < 0.8,
                       rng.choice([0, 0, 300]), _log(rng, 1, 20) - 1)
    del c["name"]
    return c


def _lens(case):
    """(tokens in the cache, new tokens) of each request: by the case alone. The longest of a range is always among them."""
    r = random.Random(case["requests"] * 1009 + case["new_max"] * 31 + case["context_max"])
    cached, new = [], []
    for b in range(case["requests"]):
        n = case["new_max"] if b == 0 else r.randint(case["new_min"], case["new_max"])
        if case["op"] == "attention" and b % 2 and case["new_max"] > 16:
            n = max(case["new_min"], 1)                        # every second request of a mixed step decodes
        total = case["context_max"] if b == 0 else _log(r, max(case["context_min"], 1), case["context_max"])
        if case["context_min"] == 0 and r.random() < 0.1:
            total = 0                                          # a request that starts with this step
        cached.append(max(total - n, 0) if case["op"] == "attention" else total)
        new.append(n)
    return cached, new


# ---- inputs ----------------------------------------------------------------------------------------------------------

_BOUNDS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)              # between the E2M1 magnitudes 0 .5 1 1.5 2 3 4 6
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _codes(x, divisor):
    """E2M1 codes and E4M3 scale bytes of f32 rows [..., D], groups of 16, in the single-precision steps of the format."""
    g = x.unflatten(-1, (-1, 16))
    d = torch.full((), divisor, device=x.device)
    s = ((g.abs().amax(-1) * d) / torch.full_like(d, 6.0)).clamp(max=448.0).to(torch.float8_e4m3fn)
    sf = s.float().unsqueeze(-1)
    v = torch.where(sf > 0, (g * d) / torch.where(sf > 0, sf, torch.ones_like(sf)), torch.zeros_like(g))
    a = v.abs()
    code = sum((a >= b) if i % 2 else (a > b) for i, b in enumerate(_BOUNDS)).to(torch.uint8)   # ties go to the even code
    code = code + (v < 0).to(torch.uint8) * 8
    return code.flatten(-2), s.view(torch.uint8)


def _pack(k, v, D):
    """Blocks [..., 18 D] of the cache from f32 rows [..., 16, D]."""
    parts = []
    for x, div, is_v in ((k, KDIV, False), (v, VDIV, True)):
        code, s = _codes(x, div)
        by = code[..., 0::2] + code[..., 1::2] * 16                                    # [..., 16, D/2]
        if is_v:
            by = by.unflatten(-2, (2, 4, 2)).unflatten(-1, (8, D // 16))               # [..., p, t, j, g, bytes]
            n = by.dim()
            by = by.permute(*range(n - 5), n - 5, n - 2, n - 4, n - 3, n - 1)          # [..., p, g, t, j, bytes]
            s = s.unflatten(-2, (2, 4, 2))
            n = s.dim()
            s = s.permute(*range(n - 4), n - 1, n - 3, n - 4, n - 2)                   # [..., group, t, p, j]
            parts += [by.flatten(-5), s.flatten(-4)]
        else:
            s = s.unflatten(-2, (2, 8)).unflatten(-1, (4, D // 64))                    # [..., h, r, t, i]
            n = s.dim()
            s = s.permute(*range(n - 4), n - 3, n - 2, n - 4, n - 1)                   # [..., r, t, h, i]
            parts += [by.flatten(-2), s.flatten(-4)]
    return torch.cat([parts[0], parts[2], parts[1], parts[3]], dim=-1)


def _unpack(blocks, D, dtype=torch.float32):
    """K and V codes times scales [..., 16, D] of blocks [..., 18 D]."""
    lut = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device=blocks.device, dtype=dtype)
    lut = torch.stack([lut.repeat(16), lut.repeat_interleave(16)], -1)                 # byte -> (low, high) nibble
    k, v = blocks[..., : 8 * D], blocks[..., 8 * D: 16 * D]
    ks, vs = blocks[..., 16 * D: 17 * D], blocks[..., 17 * D:]
    ks = ks.unflatten(-1, (8, 4, 2, D // 64))
    n = ks.dim()
    ks = ks.permute(*range(n - 4), n - 2, n - 4, n - 3, n - 1).flatten(-2).flatten(-3, -2)
    vs = vs.unflatten(-1, (D // 16, 4, 2, 2))
    n = vs.dim()
    vs = vs.permute(*range(n - 4), n - 2, n - 3, n - 1, n - 4).flatten(-4, -2)
    v = v.unflatten(-1, (2, 8, 4, 2, D // 16))
    n = v.dim()
    v = v.permute(*range(n - 5), n - 5, n - 3, n - 2, n - 4, n - 1).flatten(-2).flatten(-4, -2)
    k = k.unflatten(-1, (16, D // 2))
    out = []
    for c, s in ((k, ks), (v, vs)):
        s = s.contiguous().view(torch.float8_e4m3fn).to(dtype)
        out.append((lut[c.to(torch.int32)].flatten(-2).unflatten(-1, (-1, 16)) * s.unsqueeze(-1)).flatten(-2))
    return out


def _rope_table(case, positions):
    """[positions, rot]: cosines, then sines, from angles in 64 bits."""
    half = case["rot"] // 2
    inv = 1e6 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    a = torch.arange(positions, device=DEV, dtype=torch.float64).unsqueeze(1) * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _pages_for(cached, new, page):
    return [-(-(c + n) // page) for c, n in zip(cached, new)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": case}

    def rows(n, h, d):
        x = torch.randn(n, h, d, generator=g, device=DEV)
        return x.to(torch.bfloat16) if case.get("dtype", "bf16") == "bf16" else x

    if case["op"] == "plan":
        cached, new = _lens(case)
        page = case["page"]
        want = _pages_for(cached, new, page)
        have = [-(-c // page) for c in cached]
        spare = 7                                             # pages that are left over after the step
        total = sum(want) + spare
        ids = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        table = torch.full((len(cached), max(want) + 3), -1, dtype=torch.int32, device=DEV)
        at = torch.tensor([0] + have, device=DEV).cumsum(0)[:-1]
        h = torch.tensor(have, device=DEV).unsqueeze(1)
        col = torch.arange(table.shape[1], device=DEV).unsqueeze(0)
        table = torch.where(col < h, ids[(at.unsqueeze(1) + col).clamp(max=total - 1)], table).contiguous()
        s.update(cached=torch.tensor(cached, dtype=torch.int32, device=DEV), new=torch.tensor(new, dtype=torch.int32, device=DEV),
                 table=table, free=ids[sum(have):].contiguous(), taken=torch.zeros(1, dtype=torch.int32, device=DEV),
                 tokens=sum(new) + case["spare_rows"])
        return s

    D, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    if case["op"] in ("norm_rope", "store"):
        T, reach = case["tokens"], 40000
        s.update(q=rows(T, hq, D) * 2, k=rows(T, hkv, D) * 3, v=rows(T, hkv, D),
                 qw=torch.rand(D, generator=g, device=DEV) + 0.5, kw=torch.rand(D, generator=g, device=DEV) * 2 + 0.2,
                 rope=_rope_table(case, reach), positions=torch.randint(0, reach, (T,), generator=g, device=DEV, dtype=torch.int32),
                 q_out=torch.empty(T, hq, D, dtype=torch.bfloat16, device=DEV))
        if case["op"] == "norm_rope":
            out = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
            s.update(q_out=torch.empty(T, hq, D, dtype=out, device=DEV), k_out=torch.empty(T, hkv, D, dtype=out, device=DEV))
        else:
            page = case["page"]
            pages = -(-T // page) + 5
            s.update(cache=torch.randint(0, 256, (pages, hkv, page // 16, 18 * D), generator=g, device=DEV, dtype=torch.uint8),
                     slots=torch.randperm(pages * page, generator=g, device=DEV)[:T].to(torch.int32),
                     k_out=torch.empty(T, hkv, D, device=DEV), v_out=torch.empty(T, hkv, D, device=DEV))
        return s

    cached, new = _lens(case)
    page = case["page"]
    want = _pages_for(cached, new, page)
    total, T = sum(want) + 3, sum(new) + case["spare_rows"]
    ids = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    at = torch.tensor([0] + want, device=DEV).cumsum(0)[:-1]
    col = torch.arange(max(want) + 1, device=DEV).unsqueeze(0)
    table = torch.where(col < torch.tensor(want, device=DEV).unsqueeze(1), ids[(at.unsqueeze(1) + col).clamp(max=total - 1)],
                        torch.full((), -1, dtype=torch.int32, device=DEV)).contiguous()
    cache = torch.empty(total, hkv, page // 16, 18 * D, dtype=torch.uint8, device=DEV)
    lift = torch.exp(0.5 * torch.randn(hkv, 1, 1, D, generator=g, device=DEV))        # some key channels are larger, as in real heads
    step = max(1, (1 << 25) // (hkv * page * D))
    for p in range(0, total, step):
        n = min(step, total - p)
        shape = (n, hkv, page // 16, 16, D)
        k = torch.randn(shape, generator=g, device=DEV) * lift
        cache[p: p + n] = _pack(k, torch.randn(shape, generator=g, device=DEV), D)
    q = torch.randn(T, hq, D, generator=g, device=DEV).to(torch.bfloat16)
    cu = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    s.update(q=q, cache=cache, table=table, cu=cu, kv_lens=torch.tensor([c + n for c, n in zip(cached, new)], dtype=torch.int32, device=DEV),
             out=torch.full((T, hq, D), 0.25, dtype=torch.bfloat16, device=DEV), max_new=max(new), scale=D ** -0.5)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _plain_plan(s):
    P, T = s["case"]["page"], s["tokens"]
    c, n, table, free = s["cached"].long(), s["new"].long(), s["table"], s["free"]
    width, stock = table.shape[1], free.numel()
    have = (c + P - 1) // P
    want = torch.clamp((c + n + P - 1) // P, max=width)
    need = torch.clamp(want - have, min=0)
    at = s["taken"].long() + need.cumsum(0) - need
    col = torch.arange(width, device=DEV).unsqueeze(0)
    i = col - have.unsqueeze(1)
    src = at.unsqueeze(1) + i
    fresh = torch.where(src < stock, free[src.clamp(0, stock - 1)], torch.full_like(table, -1))
    table = torch.where((i >= 0) & (col < want.unsqueeze(1)), fresh, table)
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    kv = torch.minimum(c + n, (have + torch.minimum(need, (stock - at).clamp(min=0))) * P)
    t = torch.arange(T, device=DEV)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=c.numel() - 1)
    pos = c[b] + t - cu[b]
    page = torch.where(pos // P < width, table[b, (pos // P).clamp(max=width - 1)].long(), -torch.ones_like(pos))
    live = t < cu[-1]
    slots = torch.where(live & (page >= 0), page * P + pos % P, -torch.ones_like(pos))
    pos = torch.where(live, pos, -torch.ones_like(pos))
    used = torch.clamp(s["taken"].long() + need.sum(), max=stock)
    short = (s["taken"].long() + need.sum() > stock).int() + 2 * ((c + n + P - 1) // P > width).any().int() + 4 * (cu[-1] > T).int()
    return {"table": table, "cu": cu.int(), "kv_lens": kv.int(), "positions": pos.int(), "slots": slots.int(), "taken": used.int(), "status": short.int()}


def _rotated(x, w, s, dtype):
    """[T, H, D] normed and rotated in `dtype`."""
    case = s["case"]
    x, rot = x.to(dtype), case["rot"]
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(dtype)
    cs = s["rope"][s["positions"].long()].to(dtype).unsqueeze(1)
    cos, sin = cs[..., : rot // 2], cs[..., rot // 2:]
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if case["interleaved"] else (r[..., : rot // 2], r[..., rot // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([u, v], -1).flatten(-2) if case["interleaved"] else torch.cat([u, v], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _slot_bytes(s, D):
    """Where the bytes of each token's rows lie in the flat cache: K codes, V codes, K scales, V scales, [T, Hkv, bytes]."""
    cache = s["cache"]
    page, hkv = s["case"]["page"], cache.shape[1]
    slot = s["slots"].long()
    o, tau = slot % page, slot % 16
    base = ((((slot // page).unsqueeze(1) * hkv + torch.arange(hkv, device=DEV)) * (page // 16) + (o // 16).unsqueeze(1)) * (18 * D)).unsqueeze(-1)
    tau = tau.view(-1, 1, 1)
    p, t, j, h, r = tau // 8, tau // 2 % 4, tau % 2, tau // 8, tau % 8
    kc = tau * (D // 2) + torch.arange(D // 2, device=DEV)
    vb = torch.arange(D // 2, device=DEV)
    vc = 8 * D + (((p * 8 + vb // (D // 16)) * 4 + t) * 2 + j) * (D // 16) + vb % (D // 16)
    gr = torch.arange(D // 16, device=DEV)
    ks = 16 * D + ((r * 4 + gr // (D // 64)) * 2 + h) * (D // 64) + gr % (D // 64)
    vs = 17 * D + ((gr * 4 + t) * 2 + p) * 2 + j
    return [base + x for x in (kc, vc, ks, vs)]


def _plain_store(s):
    D = s["case"]["head_dim"]
    q = _rotated(s["q"], s["qw"], s, torch.float32).to(torch.bfloat16)
    k = _rotated(s["k"], s["kw"], s, torch.float64).float()     # its codes sit next to rounding borders
    flat = s["cache"].view(-1)
    kc, vc, ks, vs = _slot_bytes(s, D)
    back = []
    for x, div, ci, si in ((k, KDIV, kc, ks), (s["v"].float(), VDIV, vc, vs)):
        code, sc = _codes(x, div)
        flat[ci] = code[..., 0::2] + code[..., 1::2] * 16
        flat[si] = sc
    lut = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device=DEV)
    for div, ci, si in ((KDIV, kc, ks), (VDIV, vc, vs)):
        by = flat[ci].long()
        code = torch.stack([by % 16, by // 16], -1).flatten(-2)
        sc = flat[si].view(torch.float8_e4m3fn).float().repeat_interleave(16, -1)
        back.append(lut[code] * sc / torch.full((), div, device=DEV))
    return {"q": q, "k": back[0], "v": back[1]}


def _padded(s):
    """Queries of each request at [B, new, H, D], the mask of what they see [B, new, L], and each row's (request, place)."""
    case, cu, kv = s["case"], s["cu"].long(), s["kv_lens"].long()
    T, B = s["q"].shape[0], kv.numel()
    L = s["table"].shape[1] * case["page"]
    i = torch.arange(s["max_new"], device=DEV)
    n = cu[1:] - cu[:-1]
    q = s["q"][(cu[:-1].unsqueeze(1) + i).clamp(max=T - 1)]
    at = (kv - n).unsqueeze(1) + i
    j = torch.arange(L, device=DEV)
    see = (j < kv.view(B, 1, 1)) & (i < n.unsqueeze(1)).unsqueeze(2)
    if case["causal"]:
        see = see & (j <= at.unsqueeze(2))
    if case["window"]:
        see = see & (j > at.unsqueeze(2) - case["window"])
    t = torch.arange(T, device=DEV)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=B - 1)
    return q, see, b, (t - cu[b]).clamp(max=s["max_new"] - 1), t < cu[-1]


def _plain_attention(s):
    case = s["case"]
    D, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    G = hq // hkv
    q, see, b, i, live = _padded(s)
    blocks = s["cache"][s["table"].clamp(min=0).long()].transpose(1, 2).flatten(2, 3)          # [B, Hkv, L / 16, 18 D]
    k, v = (x.flatten(2, 3) for x in _unpack(blocks, D))                                       # [B, Hkv, L, D]
    B, new = q.shape[:2]
    q = q.float().view(B, new, hkv, G, D).transpose(1, 2).reshape(B, hkv, new * G, D)
    sc = (torch.matmul(q, k.transpose(2, 3)) * (s["scale"] / KDIV)).view(B, hkv, new, G, -1)
    del k
    see = see.view(B, 1, new, 1, -1)
    sc = sc.masked_fill(~see, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    del sc
    total = p.sum(-1, keepdim=True)
    v = torch.where((torch.arange(v.shape[2], device=DEV) < s["kv_lens"].view(B, 1, 1)).unsqueeze(-1), v, torch.zeros_like(v))
    o = torch.matmul(p.view(B, hkv, new * G, -1), v).view(B, hkv, new, G, D)
    o = torch.where(total > 0, o / torch.where(total > 0, total * VDIV, torch.ones_like(total)), torch.zeros_like(o))
    o = o.transpose(1, 2).reshape(B, new, hq, D)[b, i].to(torch.bfloat16)
    s["out"].copy_(torch.where(live.view(-1, 1, 1), o, s["out"]))
    return s["out"]


# ---- the package's calls ---------------------------------------------------------------------------------------------

def _own(s):
    """What a program keeps beside its inputs: the backend, the cache's handle, a step's arrays, a workspace."""
    global _backend
    from velox_inferer_b200 import Kv4Cache, Kv4Step, Sm100Backend
    if _backend is None:
        _backend = Sm100Backend(0)
    case = s["case"]
    if case["op"] == "plan":
        return {"step": Kv4Step(_backend, case["requests"], s["tokens"]), "taken": torch.zeros(1, dtype=torch.int32, device=DEV)}
    if case["op"] == "norm_rope":
        return {}
    own_ = {"cache": Kv4Cache(s["cache"], case["page"], case["head_dim"], KDIV, VDIV)}
    if case["op"] == "attention":
        own_["ws"] = _backend.kv4_workspace(case["heads"], case["kv_heads"], case["head_dim"])
    return own_


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "plan":
            return _plain_plan(s)
        if case["op"] == "norm_rope":
            dt = s["q_out"].dtype
            return {"q": _rotated(s["q"], s["qw"], s, torch.float32).to(dt), "k": _rotated(s["k"], s["kw"], s, torch.float32).to(dt)}
        return _plain_store(s) if case["op"] == "store" else _plain_attention(s)
    if "own" not in s:
        s["own"] = _own(s)
    b, o = _backend, s["own"]
    if case["op"] == "plan":
        st = o["step"]
        b.kv4_plan(s["cached"], s["new"], s["table"], s["free"], s["taken"], case["page"], st, o["taken"])
        return {"table": s["table"], "cu": st.cu, "kv_lens": st.kv_lens, "positions": st.positions, "slots": st.slots, "taken": o["taken"], "status": st.status}
    if case["op"] == "norm_rope":
        b.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["rope"], s["positions"], s["q_out"], s["k_out"], EPS, interleaved=case["interleaved"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if case["op"] == "store":
        b.qk_norm_rope_kv4(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["rope"], s["positions"], s["slots"], o["cache"], s["q_out"], EPS)
        b.kv4_rows(o["cache"], s["slots"], s["k_out"], s["v_out"])
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    b.kv4_attention(s["q"], s["out"], o["cache"], s["table"], s["cu"], s["kv_lens"], o["ws"], scale=s["scale"], causal=case["causal"],
                    window=case["window"], max_new=s["max_new"])
    return s["out"]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    if case["op"] == "plan":
        cached, new = _lens(case)
        page, T = case["page"], sum(new) + case["spare_rows"]
        fresh = sum(w - -(-c // page) for w, c in zip(_pages_for(cached, new, page), cached))
        return {"bytes": 16 * len(cached) + 8 * fresh + 8 * T + 16, "flops": 0}
    D, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    if case["op"] in ("norm_rope", "store"):
        T, e = case["tokens"], 4 if case["dtype"] == "f32" else 2
        b = T * (4 + 4 * case["rot"]) + T * hq * D * e + 8 * D
        if case["op"] == "norm_rope":
            return {"bytes": b + T * hkv * D * e + T * (hq + hkv) * D * e, "flops": 10 * T * (hq + hkv) * D}
        # k and v in, q out, codes and scales written and read back, the rows' values out in f32
        return {"bytes": b + 2 * T * hkv * D * e + T * hq * D * 2 + 4 * T + 2 * T * hkv * (2 * D * 9 // 16 + 4 * D), "flops": 10 * T * (hq + hkv) * D}
    cached, new = _lens(case)
    pairs = tokens = 0
    for c, n in zip(cached, new):
        tot = c + n
        tokens += tot - (max(0, c + 1 - case["window"]) if case["window"] else 0)
        for i in range(n):
            hi = min(tot, c + i + 1) if case["causal"] else tot
            lo = max(0, c + i + 1 - case["window"]) if case["window"] else 0
            pairs += max(0, hi - lo)
    T = sum(new)
    return {"bytes": tokens * hkv * D * 9 // 8 + 4 * T * hq * D + 4 * sum(_pages_for(cached, new, case["page"])), "flops": 4 * hq * D * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_rows(x, w, rope, positions, rot, interleaved):
    """Norm and rotation of [T, H, D] as complex products."""
    y = x.double()
    y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
    cs = rope.double()[positions.long()]
    turn = torch.complex(cs[:, : rot // 2], cs[:, rot // 2:]).unsqueeze(1)
    if interleaved:
        z = torch.complex(y[..., 0:rot:2].contiguous(), y[..., 1:rot:2].contiguous()) * turn
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    else:
        z = torch.complex(y[..., : rot // 2].contiguous(), y[..., rot // 2: rot].contiguous()) * turn
        y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
    return y


def _exact_values(x, divisor):
    """What a row's 4-bit form stands for: the nearest level of each group's grid, ties to the even code."""
    g = x.unflatten(-1, (-1, 16))
    s = (g.abs().amax(-1, keepdim=True) * divisor / 6.0).clamp(max=448.0).float().to(torch.float8_e4m3fn).double()
    v = torch.where(s > 0, g * divisor / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g))
    a = v.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    return (torch.round(a / step) * step * torch.sign(v) * s / divisor).flatten(-2)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    D, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    if case["op"] in ("norm_rope", "store"):
        q, k = (_exact_rows(s[x], s[x + "w"], s["rope"], s["positions"], case["rot"], case["interleaved"]) for x in ("q", "k"))
        if case["op"] == "norm_rope":
            return {"q": q, "k": k}
        return {"q": q, "k": _exact_values(k.float().double(), KDIV), "v": _exact_values(s["v"].double(), VDIV)}
    cached, new = _lens(case)
    out, G, row = s["out"].double(), hq // hkv, 0
    for b, (c, n) in enumerate(zip(cached, new)):
        tot = c + n
        pages = s["table"][b, : -(-tot // case["page"])].long()
        at = c + torch.arange(n, device=DEV).unsqueeze(1)
        j = torch.arange(tot, device=DEV)
        see = torch.ones(n, tot, dtype=torch.bool, device=DEV)
        if case["causal"]:
            see &= j <= at
        if case["window"]:
            see &= j > at - case["window"]
        for h in range(hkv):
            k, v = (x.flatten(0, 2)[:tot] for x in _unpack(s["cache"][pages, h], D, torch.float64))
            q = s["q"][row: row + n, h * G: (h + 1) * G].double()
            sc = torch.einsum("igd,jd->igj", q, k) * (s["scale"] / KDIV)
            sc = sc.masked_fill(~see.unsqueeze(1), float("-inf"))
            p = torch.nan_to_num(torch.softmax(sc, -1))
            out[row: row + n, h * G: (h + 1) * G] = torch.einsum("igj,jd->igd", p, v) / VDIV
            del sc, p
        row += n
    return out
