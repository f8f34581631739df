"""Operators of a served attention layer over a paged cache held in 4 bits, as a serving program calls them: the step's
tables (block tables, slots and positions from request lengths), the norms of the query and key heads with the position
rotation and the write into the cache, and the attention that reads it.

``run`` computes the plain form (elementary torch operations in 32 bits, rounded once at the end; keys that go into 4 bits
in 64, next to their codes' borders) where ``own`` is false, and calls the package's operators where it is true.
``exact`` states the same definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
GROUP = 32   # values that share a scale, along a head
TILE = 16    # positions of a cache record
EPS = 1e-6


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-a100-fastpath_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qwen_fastpath
    return qwen_fastpath


# ---- cases ----

def listed():
    return [
        # single-user speculative decode: one verified and 4 drafted tokens of one request
        {"name": "tables_b1", "kind": "tables", "B": 1, "context": 1000, "q": 5, "page": 16, "prefill": False, "pad": 0},
        # a mixed step of a busy server: decodes, prompt chunks of all lengths, idle requests, a padded token count
        {"name": "tables_b333_mixed", "kind": "tables", "B": 333, "context": 9000, "q": 512, "page": 48, "prefill": True,
         "pad": 77},
        # the 5 tokens of a verification step, 64 query heads over 8 key heads, into the 4-bit cache
        {"name": "rope_t5", "kind": "rope", "T": 5, "heads": 64, "kv_heads": 8, "D": 128, "rot": 128, "page": 16, "cache": "kv4",
         "norm": True, "offset": 0.0, "interleaved": False, "gated": False, "table": "bf16"},
        # a short odd prompt of a model with wide heads, a quarter of them rotated, queries beside their output gates
        {"name": "rope_t333_gated", "kind": "rope", "T": 333, "heads": 24, "kv_heads": 4, "D": 256, "rot": 64, "page": 48,
         "cache": "kv4", "norm": True, "offset": 1.0, "interleaved": False, "gated": True, "table": "f32"},
        # a prefill chunk into the 4-bit cache
        {"name": "rope_t2048", "kind": "rope", "T": 2048, "heads": 64, "kv_heads": 8, "D": 128, "rot": 128, "page": 64,
         "cache": "kv4", "norm": True, "offset": 0.0, "interleaved": False, "gated": False, "table": "bf16"},
        # a long odd chunk into bf16 pages, neighbouring values rotated as pairs
        {"name": "rope_t8191_pages", "kind": "rope", "T": 8191, "heads": 16, "kv_heads": 2, "D": 128, "rot": 64, "page": 16,
         "cache": "bf16", "norm": True, "offset": 0.0, "interleaved": True, "gated": False, "table": "bf16"},
        # one decoded token at a short context: latency
        {"name": "attn_1k", "kind": "attn", "B": 1, "q": 1, "ragged_q": False, "context": 1000, "heads": 64, "kv_heads": 8,
         "D": 128, "page": 16},
        # a verification step of one long request with wide heads
        {"name": "attn_verify_38k", "kind": "attn", "B": 1, "q": 3, "ragged_q": False, "context": 38000, "heads": 24,
         "kv_heads": 4, "D": 256, "page": 16},
        # a decode batch of ragged lengths
        {"name": "attn_decode_b48", "kind": "attn", "B": 48, "q": 1, "ragged_q": False, "context": 9000, "heads": 64,
         "kv_heads": 8, "D": 128, "page": 64},
        # verification of an odd batch with narrow heads, some requests too short for their first queries
        {"name": "attn_verify_b7_d64", "kind": "attn", "B": 7, "q": 4, "ragged_q": False, "context": 5000, "heads": 32,
         "kv_heads": 4, "D": 64, "page": 48},
        # prompt chunks of different lengths beside single decoded tokens in one call
        {"name": "attn_ragged_b9_d256", "kind": "attn", "B": 9, "q": 700, "ragged_q": True, "context": 4000, "heads": 24,
         "kv_heads": 4, "D": 256, "page": 16},
        # a full prefill chunk behind a cached prompt
        {"name": "attn_prefill_2048", "kind": "attn", "B": 1, "q": 2048, "ragged_q": False, "context": 8192, "heads": 64,
         "kv_heads": 8, "D": 128, "page": 64},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rope", "rope", "attn", "attn", "attn"])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if kind == "tables":
        prefill = rng.random() < 0.5
        B = _log_int(rng, 1, 333)
        return {"kind": kind, "B": B, "context": _log_int(rng, 8, 9000), "q": _log_int(rng, 2, 512) if prefill else rng.randint(1, 8),
                "page": page, "prefill": prefill, "pad": rng.choice([0, 0, rng.randint(1, 64)])}
    D = rng.choice([64, 128, 128, 256])
    if kind == "rope":
        kv = rng.choice([1, 2, 4, 5, 8])
        heads = kv * rng.randint(1, 8)
        most = 2048 * 80 * 128 // ((heads + 2 * kv) * D)
        return {"kind": kind, "T": _log_int(rng, 1, min(8192, most)), "heads": heads, "kv_heads": kv, "D": D,
                "rot": rng.choice([D, D, D // 2, D // 4]), "page": page, "cache": rng.choice(["kv4", "kv4", "bf16"]),
                "norm": rng.random() < 0.75, "offset": rng.choice([0.0, 1.0]), "interleaved": rng.random() < 0.3,
                "gated": rng.random() < 0.3, "table": rng.choice(["bf16", "f32"])}
    kv = rng.choice([1, 2, 4, 8])
    G = rng.randint(1, 8)
    case = {"kind": kind, "heads": kv * G, "kv_heads": kv, "D": D, "page": page}
    if rng.random() < 0.6:  # decode and verification
        B = _log_int(rng, 1, 48)
        most = 48 * 9000 * 8 * 128 // (B * kv * D)
        return {**case, "B": B, "q": rng.randint(1, 6), "ragged_q": rng.random() < 0.2, "context": _log_int(rng, 16, min(40000, most))}
    B = _log_int(rng, 1, 9)
    q = _log_int(rng, 8, 2048 if B == 1 else 700)
    most = int(6e11 / (4 * kv * G * D * B * q)) - q
    return {**case, "B": B, "q": q, "ragged_q": B > 1, "context": _log_int(rng, 1, max(2, min(16000, most)))}


# ---- inputs ----

def _lengths(g, B, most, least=1):
    """B lengths up to `most`, the first the longest, spread over their logarithm."""
    x = torch.rand(B, generator=g) * math.log(max(most, least + 1) / least) + math.log(least)
    n = x.exp().round().long().clamp(least, max(most, least))
    n[0] = most
    return n


def _queries(g, case):
    """New tokens of each request: the same lengths for every seed, so that outputs have one shape, in another order."""
    fixed = torch.Generator()
    fixed.manual_seed(case["B"] * 8191 + case["q"])
    B = case["B"]
    if case.get("prefill") or case.get("ragged_q"):
        q = _lengths(fixed, B, case["q"])
    elif case["kind"] == "tables":
        q = torch.randint(1, case["q"] + 1, (B,), generator=fixed)
    else:
        q = torch.full((B,), case["q"])
    if case["kind"] == "tables":
        q[torch.rand(B, generator=fixed) < 0.1] = 0  # idle requests of the batch
    q[0] = case["q"]
    q[1:] = q[1:][torch.randperm(B - 1, generator=g)]
    return q


def _pages(g, counts, page, spare=3):
    """A shuffled pool: (blocks in the pool, int32 [B, widest] tables whose entries past a request's pages are 0, the
    blocks nobody holds)."""
    total = int(counts.sum())
    order = torch.randperm(total + spare, generator=g)
    table = torch.zeros(len(counts), max(1, int(counts.max())), dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts.tolist()):
        table[b, :n] = order[at:at + n].int()
        at += n
    return total + spare, table, order[at:]


def _ceil(a, b):
    return -(-a // b)


def _e2m1(y):
    """Codes 0..15 (sign, then 0 .5 1 1.5 2 3 4 6) of y rounded to nearest even, at most 6."""
    a = y.abs()
    m = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), (torch.round(a / 2) * 2).clamp(max=6)))
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4))
    return (code + 8 * (y < 0)).to(torch.uint8)


def _quantised(x):
    """(codes uint8 [..., D], scale exponents + 127 uint8 [..., D / 32]) of bf16 values: 2^e with the block's largest
    magnitude below 7 * 2^e, from 2^-125 on."""
    f = x.float().unflatten(-1, (-1, GROUP))
    top = f.abs().amax(-1, keepdim=True)
    e = ((top.view(torch.int32) + 0x200000) >> 23).clamp(min=4) - 2
    scale = (e << 23).view(torch.float32)
    return _e2m1(f / scale).flatten(-2), e.squeeze(-1).to(torch.uint8)


def _values(codes, e):
    """The fp32 values that codes [..., D] and scale exponents [..., D / 32] stand for."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    scale = (e.int() << 23).view(torch.float32)
    return (grid[codes.long()].unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)


def _records(kc, ke, vc, ve):
    """The cache of [blocks, page, kv_heads, D] codes and [.., D / 32] scales: uint8 [blocks, kv_heads, page / 16, 17 D].  A
    record of 16 positions holds the keys' codes [position][D / 2] (the even value in the low half of a byte), the values'
    codes [D / (16 w)][4 quads of positions][16][position in the quad][w / 2] with w = min(D, 128) / 16 neighbouring values
    together, the keys' scales [D / 32][position] and the values' scales likewise."""
    n, page, hkv, D = kc.shape
    w = min(D, 128) // 16

    def tiles(t):
        return t.view(n, page // TILE, TILE, hkv, -1).permute(0, 3, 1, 2, 4)

    def halves(t):
        return t[..., 0::2] | (t[..., 1::2] << 4)

    keys = halves(tiles(kc)).reshape(n, hkv, page // TILE, -1)
    v = halves(tiles(vc)).view(n, hkv, page // TILE, 4, 4, D // (16 * w), 16, w // 2)
    values = v.permute(0, 1, 2, 5, 3, 6, 4, 7).reshape(n, hkv, page // TILE, -1)
    scales = [tiles(e).transpose(-1, -2).reshape(n, hkv, page // TILE, -1) for e in (ke, ve)]
    return torch.cat([keys, values] + scales, -1).contiguous()


def _unpacked(cache):
    """_records undone: (kc, ke, vc, ve) by [blocks, page, kv_heads, ..]."""
    n, hkv, tiles, size = cache.shape
    D = size // 17
    w = min(D, 128) // 16

    def both(t):
        return torch.stack([t & 15, t >> 4], -1).flatten(-2)

    def rows(t):
        return t.permute(0, 2, 3, 1, 4).reshape(n, tiles * TILE, hkv, -1)

    kc = rows(both(cache[..., :8 * D].reshape(n, hkv, tiles, TILE, D // 2)))
    v = cache[..., 8 * D:16 * D].reshape(n, hkv, tiles, D // (16 * w), 4, 16, 4, w // 2)
    vc = rows(both(v.permute(0, 1, 2, 4, 6, 3, 5, 7).reshape(n, hkv, tiles, TILE, D // 2)))
    ke, ve = (rows(cache[..., a:a + D // 2].reshape(n, hkv, tiles, D // GROUP, TILE).transpose(-1, -2))
              for a in (16 * D, 16 * D + D // 2))
    return kc, ke, vc, ve


def _angles(positions, rot):
    """fp32 [positions, rot]: cosines, then sines, made in 64 bits."""
    inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], -1).float()


def prepare(case, seed):
    host = torch.Generator()
    host.manual_seed(int(seed))
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    randn = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    page = case["page"]
    if case["kind"] == "tables":
        B = case["B"]
        context = _lengths(host, B, case["context"])
        q = _queries(host, case)
        held = _ceil(context, page) + (torch.rand(B, generator=host) < 0.2).long()  # some hold a page from a rejected draft
        blocks, table, free = _pages(host, held, page, int(_ceil(q, page).sum()) + B + 7)
        width = _ceil(case["context"] + case["q"], page) + 4
        wide = torch.zeros(B, width, dtype=torch.int32)
        wide[:, :table.shape[1]] = table
        return {"case": case, "context": context.int().to(DEV), "q": q.int().to(DEV), "held": held.int().to(DEV),
                "table": wide.to(DEV), "free": free.int().to(DEV),
                "count": torch.tensor([len(free)], dtype=torch.int32, device=DEV), "tokens": int(q.sum()) + case["pad"]}
    H, hkv, D = case["heads"], case["kv_heads"], case["D"]
    channels = 1 + 6 * (torch.rand(hkv, D, device=DEV, generator=g) < 0.03)  # a few channels of a trained model's keys are large
    if case["kind"] == "rope":
        T, wide = case["T"], 2 if case["gated"] else 1
        qkv = randn(T, (wide * H + 2 * hkv) * D)
        qkv *= torch.exp(0.5 * randn(T, 1))
        qkv[:, wide * H * D:(wide * H + hkv) * D] *= channels.flatten()
        qkv = qkv.to(torch.bfloat16)
        q, k, v = qkv.split([wide * H * D, hkv * D, hkv * D], -1)
        first = int(torch.randint(0, 30000, (1,), generator=host))
        blocks = _ceil(T, page) + 2
        order = torch.randperm(blocks, generator=host)
        at = torch.arange(T)
        slots = order[at // page] * page + at % page
        if T > 8:
            slots[-2:] = -1  # the padding of a captured batch
        weight = lambda: (1 - case["offset"] + 0.2 * randn(D)).to(torch.bfloat16) if case["norm"] else None  # noqa: E731
        table = _angles(first + T, case["rot"])
        st = {"case": case, "q": q.view(T, H, -1)[..., :D], "k": k.view(T, hkv, D), "v": v.view(T, hkv, D),
              "q_weight": weight(), "k_weight": weight(), "positions": (first + at).to(DEV), "slots": slots.to(DEV),
              "table": table if case["table"] == "f32" else table.to(torch.bfloat16)}
        if case["cache"] == "kv4":
            st["cache"] = torch.zeros(blocks, hkv, page // TILE, 17 * D, dtype=torch.uint8, device=DEV)
        else:
            st["k_pages"] = torch.zeros(blocks, page, hkv, D, dtype=torch.bfloat16, device=DEV)
            st["v_pages"] = torch.zeros_like(st["k_pages"])
        return st
    B = case["B"]
    q = _queries(host, case)
    context = _lengths(host, B, case["context"])
    seq = context + q
    if B > 4:
        seq[1] = min(2, int(q[1]) - 1)  # shorter than its queries: the first of them see nothing
    blocks, table, _ = _pages(host, _ceil(seq, page), page)
    k = (randn(blocks, page, hkv, D) * channels).to(torch.bfloat16)
    v = (randn(blocks, page, hkv, D) * torch.exp(0.5 * randn(blocks, page, hkv, 1))).to(torch.bfloat16)
    cu = torch.cat([torch.zeros(1, dtype=torch.long), q.cumsum(0)])
    return {"case": case, "query": randn(int(q.sum()), H, D).to(torch.bfloat16), "cache": _records(*_quantised(k), *_quantised(v)),
            "seq": seq.int().to(DEV), "table": table.to(DEV), "cu": cu.int().to(DEV), "max_q": int(q.max()),
            "scale": D ** -0.5}


# ---- one pass ----

def _plain_tables(st):
    page, T = st["case"]["page"], st["tokens"]
    seq = st["context"] + st["q"]
    cu = torch.cat([torch.zeros_like(seq[:1]), st["q"].cumsum(0).int()])
    pages = (seq + page - 1) // page
    need = (pages - st["held"]).clamp(min=0)
    before = need.cumsum(0) - need
    j = torch.arange(st["table"].shape[1], device=DEV) - st["held"][:, None]
    taken = (j >= 0) & (j < need[:, None])
    place = (st["count"] - 1 - before[:, None] - j).clamp(0, len(st["free"]) - 1)
    table = torch.where(taken, st["free"][place], st["table"])
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu, t.int(), right=True) - 1
    inside = t < cu[-1]
    b = b.clamp(max=len(seq) - 1)
    pos = torch.where(inside, st["context"][b] + t - cu[b], 0)
    slots = torch.where(inside, table[b, pos // page].long() * page + pos % page, -1)
    return {"cu_q": cu, "seq_lens": seq, "positions": pos.long(), "slots": slots, "held": st["held"] + need,
            "free_count": st["count"] - need.sum().int(), "block_table": table}


def _rotated(n, c, s, interleaved):
    rot = 2 * c.shape[-1]
    r, rest = n[..., :rot], n[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    x, y = a * c - b * s, b * c + a * s
    r = torch.stack([x, y], -1).flatten(-2) if interleaved else torch.cat([x, y], -1)
    return torch.cat([r, rest], -1)


def _plain_rope(st):
    case = st["case"]
    page = case["page"]
    cs = st["table"][st["positions"]][:, None]
    half = cs.shape[-1] // 2

    def head(x, w, wide):
        x = x.to(wide)
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (case["offset"] + w.to(wide))
        return _rotated(x, cs[..., :half].to(wide), cs[..., half:].to(wide), case["interleaved"]).to(torch.bfloat16)

    q = head(st["q"], st["q_weight"], torch.float32)
    k = head(st["k"], st["k_weight"], torch.float64 if case["cache"] == "kv4" else torch.float32)
    v, slots = st["v"], st["slots"]
    if case["cache"] == "kv4":
        k, v = (torch.where(slots[:, None, None] >= 0, _values(*_quantised(x)), 0).to(torch.bfloat16) for x in (k, v))
        return q, k, v
    kept = slots >= 0
    st["k_pages"].flatten(0, 1)[slots[kept]] = k[kept]
    st["v_pages"].flatten(0, 1)[slots[kept]] = v[kept]
    return q, st["k_pages"], st["v_pages"]


def _plain_attn(st):
    case = st["case"]
    H, hkv, D, B, Q = case["heads"], case["kv_heads"], case["D"], case["B"], st["max_q"]
    kc, ke, vc, ve = _unpacked(st["cache"])
    table = st["table"].long()
    k, v = (_values(c, e)[table].flatten(1, 2).transpose(1, 2) for c, e in ((kc, ke), (vc, ve)))  # [B, hkv, L, D]
    L = k.shape[2]
    # the batch's queries padded to the longest: row i of request b
    i = torch.arange(Q, device=DEV)
    n = st["cu"].diff()
    row = (st["cu"][:-1, None] + torch.minimum(i, (n - 1).clamp(min=0)[:, None])).clamp(max=len(st["query"]) - 1)
    q = st["query"].float()[row].view(B, Q, hkv, H // hkv, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * st["scale"]
    last = (st["seq"] - n)[:, None] + i  # the last position each query sees
    seen = torch.arange(L, device=DEV) <= last[..., None]  # [B, Q, L]
    s = s.view(B, hkv, H // hkv, Q, L).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s -= torch.where(top == -math.inf, 0.0, top)
    p = s.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, -1, L), v.contiguous()).view(B, hkv, H // hkv, Q, D) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(B * Q, H, D)
    return o[(i < n[:, None]).flatten()].to(torch.bfloat16)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"tables": _plain_tables, "rope": _plain_rope, "attn": _plain_attn}[kind](state)
    qf = _package()
    if kind == "tables":
        t = qf.step_tables(state["context"], state["q"], state["held"], state["table"], state["free"], state["count"],
                           case["page"], state["tokens"])
        return {"cu_q": t.cu_q, "seq_lens": t.seq_lens, "positions": t.positions, "slots": t.slots, "held": t.held,
                "free_count": t.free_count, "block_table": state["table"]}
    if kind == "rope":
        cache = state["cache"] if case["cache"] == "kv4" else (state["k_pages"], state["v_pages"])
        q, _ = qf.qk_norm_rope(state["q"], state["k"], state["positions"], state["table"], state["q_weight"], state["k_weight"],
                               value=state["v"], cache=cache, slots=state["slots"], eps=EPS, weight_offset=case["offset"],
                               interleaved=case["interleaved"])
        if case["cache"] == "kv4":
            k, v = qf.kv4_load(cache, state["slots"])
            return q, k, v
        return q, state["k_pages"], state["v_pages"]
    if case["ragged_q"]:
        return qf.kv4_attention(state["query"], state["cache"], state["seq"], state["table"], state["scale"], cu_q=state["cu"],
                                max_q=state["max_q"])
    return qf.kv4_attention(state["query"], state["cache"], state["seq"], state["table"], state["scale"], q_len=case["q"])


# ---- what a pass cannot do without ----

def _spread(most, least=1):
    """The mean of _lengths' distribution."""
    most = max(most, least + 1)
    return (most - least) / math.log(most / least)


def work(case):
    if case["kind"] == "tables":
        B, page = case["B"], case["page"]
        tokens = case["q"] + (B - 1) * 0.9 * (_spread(case["q"]) if case["prefill"] else (case["q"] + 1) / 2) + case["pad"]
        return {"bytes": int(4 * (5 * B + 2) + 16 * tokens + 8 * tokens / page), "flops": int(4 * tokens)}
    H, hkv, D = case["heads"], case["kv_heads"], case["D"]
    if case["kind"] == "rope":
        T = case["T"]
        kept = T - 2 if T > 8 else T
        cache = 2 * hkv * D * (17 / 32 if case["cache"] == "kv4" else 2)
        angles = T * case["rot"] * (4 if case["table"] == "f32" else 2)
        return {"bytes": int(T * ((4 * H + 4 * hkv) * D + 16) + kept * cache + angles), "flops": T * (H + hkv) * (4 * D + 3 * case["rot"])}
    B, q, context = case["B"], case["q"], case["context"]
    n = q + (B - 1) * (_spread(q) if case["ragged_q"] else q)
    positions = context + (B - 1) * _spread(context) + n
    seen = q * (context + q / 2) + (B - 1) * (n - q) / max(1, B - 1) * (_spread(context) + (n - q) / max(1, B - 1) / 2)
    return {"bytes": int(positions * hkv * D * 2 * 17 / 32 + 4 * n * H * D), "flops": int(4 * H * D * seen)}


# ---- the definitions in 64 bits ----

def _grid64(x):
    """bf16 x as the values of its 4-bit form, from the definition: the nearest of the grid's points, the one with the even
    code among two."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for d in range(0, x.shape[-1], GROUP):
        part = x[..., d:d + GROUP].double()
        top = part.abs().amax(-1, keepdim=True)
        scale = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1e-300) / 7)) - 1).clamp(min=2.0 ** -125)
        scale = torch.where(top >= 14 * scale, 4 * scale, torch.where(top >= 7 * scale, 2 * scale, scale)).clamp(min=2.0 ** -125)
        away = (part.abs() / scale)[..., None] - grid
        off = away.abs() + torch.tensor([0, 1e-9] * 4, dtype=torch.float64, device=x.device)
        out[..., d:d + GROUP] = grid[off.argmin(-1)] * torch.sign(part) * scale
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "tables":
        return None
    H, hkv, D, page = case["heads"], case["kv_heads"], case["D"], case["page"]
    if case["kind"] == "rope":
        T, rot = case["T"], case["rot"]
        i = torch.arange(rot // 2, device=DEV)
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
        cs = st["table"].double().index_select(0, st["positions"])
        turn = torch.complex(cs[:, :rot // 2], cs[:, rot // 2:])[:, None]

        def head(x, w):
            x = x.double().clone()
            if w is not None:
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * (w.double() + case["offset"])
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            return x

        q, k, v = head(st["q"], st["q_weight"]), head(st["k"], st["k_weight"]), st["v"]
        kept = (st["slots"] >= 0).nonzero()[:, 0]
        if case["cache"] == "kv4":
            parts = []
            for x in (k.to(torch.bfloat16), v):
                y = torch.zeros(T, hkv, D, dtype=torch.float64, device=DEV)
                y[kept] = _grid64(x[kept])
                parts.append(y)
            return q, *parts
        pages = []
        for x in (k, v.double()):
            y = torch.zeros(st["k_pages"].shape, dtype=torch.float64, device=DEV)
            y[st["slots"][kept] // page, st["slots"][kept] % page] = x[kept]
            pages.append(y)
        return q, *pages
    G = H // hkv
    cu, seq = st["cu"].tolist(), st["seq"].tolist()
    out = torch.zeros(len(st["query"]), H, D, dtype=torch.float64, device=DEV)
    codes = st["cache"].view(-1, hkv, page // TILE, 17 * D)
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    lut = torch.cat([lut, -lut])
    p16, d = torch.arange(TILE, device=DEV)[:, None], torch.arange(D, device=DEV)
    w = min(D, 128) // 16
    at_key = p16 * (D // 2) + d // 2
    in_half = d % (16 * w)
    at_value = 8 * D + d // (16 * w) * (128 * w) + (((p16 // 4) * 16 + in_half // w) * 4 + p16 % 4) * (w // 2) + in_half % w // 2
    at_scale = 16 * D + d // GROUP * TILE + p16
    for b in range(case["B"]):
        n, L = cu[b + 1] - cu[b], seq[b]
        if n == 0 or L == 0:
            continue
        ids = st["table"][b, :_ceil(L, page)].long()
        last = L - n + torch.arange(n, device=DEV)
        for h in range(hkv):
            r = codes[ids, h].flatten(0, 1)  # [records, 17 D]
            kv = []
            for at, scale in ((at_key, at_scale), (at_value, at_scale + D // 2)):
                nibble = (r[:, at] >> (4 * (d % 2))) & 15
                kv.append((lut[nibble.long()] * torch.exp2(r[:, scale].double() - 127)).flatten(0, 1)[:L])
            q = st["query"][cu[b]:cu[b + 1], h * G:(h + 1) * G].double()
            s = torch.mm(q.reshape(n * G, D), kv[0].t().contiguous()).view(n, G, L) * st["scale"]
            s.masked_fill_(torch.arange(L, device=DEV) > last[:, None, None], -math.inf)
            weight = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            out[cu[b]:cu[b + 1], h * G:(h + 1) * G] = torch.mm(weight.view(n * G, L), kv[1]).view(n, G, D)
    return out
