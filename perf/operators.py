"""Operators of a block-scaled FP8 checkpoint's feed-forward, as a serving program calls them: the matrix product with
e4m3 weights and one fp32 scale for each 128 x 128 block, the norms around a block with its gate and residual scale, and a
whole mixture-of-experts layer for a few tokens.

``run`` computes the plain form (elementary torch operations in 32 bits, rounded once at the end) where ``own`` is false,
and calls the package's operators where it is true.  ``exact`` states the same definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
BLOCK = 128          # values a scale covers, in each direction of a weight and along a token's row
E4M3_MAX = 448.0
DECODE_ROWS = 16     # up to here the product keeps bf16 activations; above, they are quantised per token and block


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-a100-fastpath_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qwen_fastpath
    return qwen_fastpath


# ---- cases ----

def listed():
    return [
        # the smallest product: one token of single-user decode through a square projection
        {"name": "linear_m1", "kind": "linear", "M": 1, "N": 5120, "K": 5120, "layout": "tiled", "bias": False},
        # the widest projection of a dense layer at a verification step's width (1 verified + 4 draft tokens)
        {"name": "linear_m5_wide", "kind": "linear", "M": 5, "N": 34816, "K": 5120, "layout": "tiled", "bias": False},
        # the longest sum of that layer at the largest decode batch, weights kept in the checkpoint's layout
        {"name": "linear_m16_rows", "kind": "linear", "M": 16, "N": 5120, "K": 17408, "layout": "rowmajor", "bias": False},
        # a tensor-parallel shard of odd size: channels and k that end inside a block, a batch above the decode width
        {"name": "linear_m77_ragged", "kind": "linear", "M": 77, "N": 2500, "K": 2112, "layout": "rowmajor", "bias": True},
        # a short prompt of odd length through an output projection
        {"name": "linear_m333", "kind": "linear", "M": 333, "N": 5120, "K": 8192, "layout": "tiled", "bias": False},
        # a full prefill chunk through the widest projection
        {"name": "linear_m2048", "kind": "linear", "M": 2048, "N": 34816, "K": 5120, "layout": "tiled", "bias": False},
        # the residual step of one decoded token: a norm after the block, a norm before the next
        {"name": "norm_m1", "kind": "norm", "M": 1, "N": 5120, "post": True, "gate": "none", "act": "none",
         "alpha": 1.0, "wide": False},
        # a prefill chunk with a per-channel gate, a residual scale and an fp32 residual stream
        {"name": "norm_m2048", "kind": "norm", "M": 2048, "N": 5120, "post": True, "gate": "channel", "act": "none",
         "alpha": 0.35, "wide": True},
        # a long odd batch gated value by value (a sigmoid output gate), no norm after the block
        {"name": "norm_m8191_gated", "kind": "norm", "M": 8191, "N": 2568, "post": False, "gate": "full", "act": "sigmoid",
         "alpha": 1.0, "wide": False},
        # one decoded token through a layer of 64 experts
        {"name": "moe_t1", "kind": "moe", "T": 1, "E": 64, "k": 8, "H": 2048, "I": 768, "renorm": True, "logits": "f32"},
        # an odd batch through wide experts, bf16 router, weights of the whole softmax, k that ends inside a block
        {"name": "moe_t7_odd", "kind": "moe", "T": 7, "E": 60, "k": 4, "H": 2112, "I": 1344, "renorm": False,
         "logits": "bf16"},
        # the widest batch: nearly every expert is read
        {"name": "moe_t16", "kind": "moe", "T": 16, "E": 128, "k": 8, "H": 2048, "I": 768, "renorm": True, "logits": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "norm", "moe", "moe"])
    if kind == "linear":
        M = rng.randint(1, DECODE_ROWS) if rng.random() < 0.5 else _log_int(rng, DECODE_ROWS + 1, 2048)
        return {"kind": kind, "M": M, "N": _log_int(rng, 200, 34816), "K": 64 * _log_int(rng, 2, 80),
                "layout": rng.choice(["tiled", "tiled", "rowmajor"]), "bias": rng.random() < 0.3}
    if kind == "norm":
        return {"kind": kind, "M": _log_int(rng, 1, 8192), "N": 8 * _log_int(rng, 8, 1280), "post": rng.random() < 0.7,
                "gate": rng.choice(["none", "channel", "token", "full"]), "act": rng.choice(["none", "sigmoid"]),
                "alpha": round(rng.uniform(0.1, 1.5), 3), "wide": rng.random() < 0.4}
    E = _log_int(rng, 4, 160)
    return {"kind": kind, "T": rng.randint(1, 16), "E": E, "k": rng.randint(1, min(8, E)), "H": 64 * rng.randint(8, 40),
            "I": 64 * _log_int(rng, 2, 24), "renorm": rng.random() < 0.5, "logits": rng.choice(["f32", "bf16"])}


# ---- inputs ----

def _blocks(n):
    return -(-n // BLOCK)


def _weight(g, N, K):
    """e4m3 [N, K] and fp32 [ceil(N / 128), ceil(K / 128)] scales, as a checkpoint's quantiser makes them: the block's
    largest magnitude lands on 448.  Rows differ in size by a log-normal factor."""
    w = torch.randn(N, K, device=DEV, generator=g)
    w *= 0.02 * torch.exp(0.5 * torch.randn(N, 1, device=DEV, generator=g))
    nb, kb = _blocks(N), _blocks(K)
    padded = torch.zeros(nb * BLOCK, kb * BLOCK, device=DEV)
    padded[:N, :K] = w
    s = padded.view(nb, BLOCK, kb, BLOCK).abs().amax(dim=(1, 3)) / E4M3_MAX
    q = (padded.view(nb, BLOCK, kb, BLOCK) / s[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:N, :K]
    return q.contiguous().to(torch.float8_e4m3fn), s


def _tiles(q):
    """The load-time image of a [N, K] weight: 1 KiB tiles of 16 channels x 64 k, a tile's byte 16 (16 g + r) + i channel
    r, k 16 g + i; channels past N are zero."""
    N, K = q.shape
    rows = torch.zeros(-(-N // 16) * 16, K, dtype=torch.uint8, device=q.device)
    rows[:N] = q.view(torch.uint8)
    return rows.view(-1, 16, K // 64, 4, 16).permute(0, 2, 3, 1, 4).contiguous().view(-1).view(torch.float8_e4m3fn)


def _activations(g, M, K):
    """bf16 rows with a few channels far larger than the rest, as a trained model's are."""
    x = torch.randn(M, K, device=DEV, generator=g)
    x *= 1 + 30 * (torch.rand(1, K, device=DEV, generator=g) < 0.004)
    return x.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    kind = case["kind"]
    if kind == "linear":
        q, s = _weight(g, case["N"], case["K"])
        return {"case": case, "x": _activations(g, case["M"], case["K"]), "q": q, "s": s,
                "image": _tiles(q) if case["layout"] == "tiled" else None,
                "bias": torch.randn(case["N"], device=DEV, generator=g).to(torch.bfloat16) if case["bias"] else None}
    if kind == "norm":
        M, N = case["M"], case["N"]
        shape = {"none": None, "channel": (N,), "token": (M, 1), "full": (M, N)}[case["gate"]]
        weight = lambda: (1 + 0.2 * torch.randn(N, device=DEV, generator=g)).to(torch.bfloat16)  # noqa: E731
        residual = 4 * torch.randn(M, N, device=DEV, generator=g)
        return {"case": case, "x": _activations(g, M, N), "residual": residual if case["wide"] else residual.to(torch.bfloat16),
                "post": weight() if case["post"] else None, "pre": weight(),
                "gate": torch.randn(*shape, device=DEV, generator=g).to(torch.bfloat16) if shape else None}
    T, E, H, I = case["T"], case["E"], case["H"], case["I"]
    logits = 2 * torch.randn(T, E, device=DEV, generator=g)
    w13, s13, w2, s2 = [], [], [], []
    for _ in range(E):
        (gate, s_gate), (up, s_up), (down, s_down) = _weight(g, I, H), _weight(g, I, H), _weight(g, H, I)
        w13.append(torch.cat([gate.view(torch.uint8), up.view(torch.uint8)]))
        s13.append(torch.cat([s_gate, s_up]))
        w2.append(down.view(torch.uint8))
        s2.append(s_down)
    w13 = torch.stack(w13).view(torch.float8_e4m3fn)
    w2 = torch.stack(w2).view(torch.float8_e4m3fn)
    return {"case": case, "x": _activations(g, T, H), "logits": logits if case["logits"] == "f32" else logits.to(torch.bfloat16),
            "w13": w13, "s13": torch.stack(s13), "w2": w2, "s2": torch.stack(s2),
            "image13": _tiles(w13.view(E * 2 * I, H)), "image2": _tiles(w2.view(E * H, I))}


# ---- one pass ----

def _widened(q, s):
    """fp32 weights of e4m3 values [..., N, K] and block scales [..., ceil(N / 128), ceil(K / 128)]."""
    N, K = q.shape[-2:]
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., :N, :].repeat_interleave(BLOCK, -1)[..., :K]


def _token_blocks(x):
    """x rounded to e4m3 with one scale for each token and block of 128 values, as the fp32 values that stands for."""
    M, K = x.shape
    kb = _blocks(K)
    rows = torch.zeros(M, kb * BLOCK, device=x.device)
    rows[:, :K] = x
    rows = rows.view(M, kb, BLOCK)
    s = rows.abs().amax(-1, keepdim=True) / E4M3_MAX
    q = torch.where(s > 0, rows / s, torch.zeros_like(rows)).to(torch.float8_e4m3fn).float()
    return (q * s).view(M, kb * BLOCK)[:, :K]


def _plain_linear(st):
    x = st["x"].float()
    a = x if x.shape[0] <= DECODE_ROWS else _token_blocks(x)
    y = a @ _widened(st["q"], st["s"]).t()
    return (y if st["bias"] is None else y + st["bias"].float()).to(torch.bfloat16)


def _plain_norm(st, eps=1e-6):
    case, p, y = st["case"], st["x"].float(), st["residual"].float()
    if st["post"] is not None:
        p = p * torch.rsqrt((p * p).mean(-1, keepdim=True) + eps) * st["post"].float()
    if st["gate"] is not None:
        g = st["gate"].float()
        p = p * (1 / (1 + torch.exp(-g)) if case["act"] == "sigmoid" else g)
    y = y + case["alpha"] * p
    h = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * st["pre"].float()
    return y.to(st["residual"].dtype), h.to(torch.bfloat16)


def _routing(logits, k, renorm):
    """The k experts of each token (the largest logits, the lowest index first among equal ones) and their weights."""
    value, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids = order[:, :k]
    e = torch.exp(value - value[:, :1])
    return ids, e[:, :k] / (e[:, :k] if renorm else e).sum(-1, keepdim=True)


def _plain_moe(st):
    case, x = st["case"], st["x"].float()
    I = case["I"]
    ids, c = _routing(st["logits"].float(), case["k"], case["renorm"])
    gate = _widened(st["w13"][:, :I][ids], st["s13"][:, :_blocks(I)][ids])
    up = _widened(st["w13"][:, I:][ids], st["s13"][:, _blocks(I):][ids])
    column = x[:, None, :, None]
    a, b = (gate @ column).squeeze(-1), (up @ column).squeeze(-1)
    h = a / (1 + torch.exp(-a)) * b
    out = (_widened(st["w2"][ids], st["s2"][ids]) @ h[..., None]).squeeze(-1)
    return (c[..., None] * out).sum(1).to(torch.bfloat16)


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"linear": _plain_linear, "norm": _plain_norm, "moe": _plain_moe}[kind](state)
    qf = _package()
    case = state["case"]
    if kind == "linear":
        w = state["image"] if state["image"] is not None else state["q"].t()
        return qf.fp8_linear(state["x"], w, state["s"], state["bias"], out_features=case["N"])
    if kind == "norm":
        return qf.block_norm_rows(state["x"], state["residual"], state["post"], state["pre"], gate=state["gate"],
                                  gate_act=case["act"], alpha=case["alpha"], eps=1e-6)
    return qf.moe_few_tokens(state["x"], state["logits"], state["image13"], state["s13"], state["image2"], state["s2"],
                             case["k"], renormalize=case["renorm"])


# ---- what a pass cannot do without ----

def work(case):
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K + 4 * _blocks(N) * _blocks(K) + 2 * M * K + 2 * M * N + (2 * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    if case["kind"] == "norm":
        M, N = case["M"], case["N"]
        gate = {"none": 0, "channel": 2 * N, "token": 2 * M, "full": 2 * M * N}[case["gate"]]
        return {"bytes": M * N * (2 + 2 + (8 if case["wide"] else 4)) + 2 * N * (1 + case["post"]) + gate, "flops": 12 * M * N}
    T, E, k, H, I = case["T"], case["E"], case["k"], case["H"], case["I"]
    experts = E * (1 - (1 - k / E) ** T)  # distinct ones, expected for even routing
    scales = 4 * (2 * _blocks(I) * _blocks(H) + _blocks(H) * _blocks(I))
    return {"bytes": int(experts * (3 * I * H + scales) + 4 * T * H + T * E * (4 if case["logits"] == "f32" else 2)),
            "flops": 6 * T * k * H * I}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    st = prepare(case, seed)
    at = lambda n: torch.arange(n, device=DEV) // BLOCK  # noqa: E731  (the block of each row or column)
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x, w = st["x"].double(), st["q"].double()
        w *= st["s"].double()[at(N)][:, at(K)]
        if M > DECODE_ROWS:
            top = torch.zeros(M, _blocks(K), dtype=torch.float64, device=DEV)
            top.scatter_reduce_(1, at(K).expand(M, K), x.abs(), "amax")
            scale = (top / 448).float().double()[:, at(K)]  # the scale is an fp32 number
            ratio = torch.where(scale > 0, x / scale, 0.0)
            x = ratio.float().to(torch.float8_e4m3fn).double() * scale
        y = torch.mm(x, w.T)
        return y if st["bias"] is None else y + st["bias"].double()
    if case["kind"] == "norm":
        rms = lambda v: v / torch.sqrt(v.pow(2).sum(1, keepdim=True) / case["N"] + 1e-6)  # noqa: E731
        p = st["x"].double()
        if case["post"]:
            p = rms(p) * st["post"].double()
        if st["gate"] is not None:
            g = st["gate"].double()
            p = p * (torch.sigmoid(g) if case["act"] == "sigmoid" else g)
        y = st["residual"].double() + p * case["alpha"]
        return y, rms(y) * st["pre"].double()
    T, E, k, H, I = case["T"], case["E"], case["k"], case["H"], case["I"]
    x, logits = st["x"].double(), st["logits"].double()
    y = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    above = (logits[:, None, :] > logits[:, :, None]) | (
        (logits[:, None, :] == logits[:, :, None]) & (torch.arange(E, device=DEV) < torch.arange(E, device=DEV)[:, None]))
    chosen = above.sum(-1) < k
    c = torch.softmax(logits, -1)
    if case["renorm"]:
        c = c / (c * chosen).sum(-1, keepdim=True)
    for e in range(E):
        rows = chosen[:, e].nonzero()[:, 0]
        s13, w13 = st["s13"][e].double(), st["w13"][e].double()
        g = x[rows] @ (w13[:I] * s13[:_blocks(I)][at(I)][:, at(H)]).T
        u = x[rows] @ (w13[I:] * s13[_blocks(I):][at(I)][:, at(H)]).T
        down = st["w2"][e].double() * st["s2"][e].double()[at(H)][:, at(I)]
        y[rows] += c[rows, e][:, None] * ((g * torch.sigmoid(g) * u) @ down.T)
    return y
