"""Cases for the operators of a mixture-of-experts block in block FP8: what is timed and what is compared.

  route    top-k of the router's logits, softmax weights, and the dispatch plan: rows sorted by expert
  gate_up  matrix products grouped by expert, ragged row counts: gate_up + SiLU(gate) * up + e4m3 group quant
  down     matrix products grouped by expert, ragged row counts: e4m3 rows -> bf16 rows
  block    the block's end: weighted sum of each token's expert rows (or a dense output), norm after the block,
           gate, residual scale, and the norm before the next block with its e4m3 group quant

`own` false: plain torch in 32 bits. `own` true: the calls a user makes of fp8_hand_b200.
"""
import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------ the cases
def _route(name, T, E, k, dtype="bf16", renormalize=True, begin=0, count=0, masked=0.0):
    """count 0: every expert is local. masked: share of the tokens that are padding (all logits -inf)."""
    return {"name": name, "op": "route", "T": T, "E": E, "k": k, "dtype": dtype, "renormalize": renormalize,
            "begin": begin, "count": count or E, "masked": masked}


def _gate_up(name, T, E, k, H, I, tiled=True, skew=0.5):
    return {"name": name, "op": "gate_up", "T": T, "E": E, "k": k, "H": H, "I": I, "tiled": tiled, "skew": skew}


def _down(name, T, E, k, H, I, tiled=True, skew=0.5):
    return {"name": name, "op": "down", "T": T, "E": E, "k": k, "H": H, "I": I, "tiled": tiled, "skew": skew}


def _block(name, T, k, H, post=True, gate="channel", wide=False):
    """k 0: a dense output. gate: none, channel [H], token [T, 1] or full [T, H]. wide: fp32 residual."""
    return {"name": name, "op": "block", "T": T, "k": k, "H": H, "post": post, "gate": gate, "wide": wide}


def listed():
    return [
        # one token being decoded: latency alone
        _route("route_1", 1, 64, 8),
        # a ragged batch on one of two expert-parallel ranks, fp32 logits, a few padding tokens of a captured graph
        _route("route_333_half_local", 333, 160, 6, dtype="f32", renormalize=False, begin=80, count=80, masked=0.05),
        # a full prefill chunk
        _route("route_8192", 8192, 128, 8),
        # one token: eight experts with a row each, the weights' read is everything
        _gate_up("gate_up_1", 1, 64, 8, 5120, 1024),
        # a decode batch of odd size: nearly every expert has a few rows
        _gate_up("gate_up_61", 61, 64, 8, 5120, 1024),
        # a short prefill, as many weights as arithmetic; row-major weights, as loaded without a pre-pack
        _gate_up("gate_up_1000", 1000, 64, 8, 5120, 1024, tiled=False),
        # a full prefill chunk: tensor bound
        _gate_up("gate_up_8192", 8192, 64, 8, 5120, 1024),
        # a small decode batch
        _down("down_5", 5, 64, 8, 5120, 1024),
        # speculative verify of a batch, many small experts
        _down("down_240", 240, 128, 6, 2048, 768),
        # a full prefill chunk
        _down("down_8192", 8192, 64, 8, 5120, 1024),
        # one token's end of the block
        _block("block_1", 1, 8, 5120),
        # a full prefill chunk's, with a gate per token
        _block("block_8192", 8192, 8, 5120, gate="token"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _log_mult(rng, lo, hi, step):
    return max(lo, min(hi, _log_int(rng, lo, hi) // step * step))


def draw(rng):
    op = rng.choice(["route", "gate_up", "down", "block"])
    T, k = _log_int(rng, 1, 8192), rng.randint(1, 8)
    if op == "route":
        E = rng.randint(max(8, k), 160)
        count = rng.choice([E, max(1, E // 2), max(1, E // 4)])
        return {"op": op, "T": T, "E": E, "k": k, "dtype": rng.choice(["bf16", "f32"]), "renormalize": rng.random() < 0.5,
                "begin": rng.randint(0, E - count), "count": count, "masked": rng.choice([0.0, 0.1])}
    if op == "block":
        return {"op": op, "T": T, "k": rng.choice([0, k]), "H": _log_mult(rng, 1024, 5120, BLOCK), "post": rng.random() < 0.7,
                "gate": rng.choice(["none", "channel", "token", "full"]), "wide": rng.random() < 0.3}
    E = _log_int(rng, 8, 160)
    H, I = _log_mult(rng, 1024, 5120, BLOCK), _log_mult(rng, 256, 2048, BLOCK)
    while E * H * I > 64 * 5120 * 1024:
        E //= 2
    k = min(k, E)
    while T * k * H * I > 8192 * 8 * 5120 * 1024:
        T //= 2
    return {"op": op, "T": T, "E": E, "k": k, "H": H, "I": I, "tiled": rng.random() < 0.5, "skew": rng.choice([0.0, 0.5, 1.0])}


def work(case):
    T = case["T"]
    if case["op"] == "route":
        E, R = case["E"], T * case["k"]
        logits = T * E * (2 if case["dtype"] == "bf16" else 4)
        return {"bytes": logits + 4 * (4 * R + case["count"] + 1), "flops": 4.0 * T * E}
    H = case["H"]
    if case["op"] == "block":
        rows = max(1, case["k"])
        res = 2 * (4 if case["wide"] else 2)
        gate = {"none": 0, "channel": 2 * H, "token": 2 * T, "full": 2 * T * H}[case["gate"]]
        b = T * H * (2 * rows + res + 1) + 4 * T * (H // BLOCK) + gate + 4 * H + 8 * T * case["k"]
        return {"bytes": b, "flops": float(T * H * (2 * rows + 12))}
    E, k, I = case["E"], case["k"], case["I"]
    R = T * k
    active = E * (1.0 - (1.0 - k / E) ** T)  # experts with a row, in expectation over even routing
    N, K = (2 * I, H) if case["op"] == "gate_up" else (H, I)
    b = active * N * (K + 4 * K / BLOCK / BLOCK)
    if case["op"] == "gate_up":
        b += T * (K + K // 32) + R * (I + I // 32) + 4 * R
    else:
        b += R * (K + K // 32) + 2 * R * N
    return {"bytes": b, "flops": 2.0 * R * N * K}


# ------------------------------------------------------------------ inputs
def _quant_rows(x):
    """Groups of 128 along a row: (e4m3, fp32 scales)."""
    g = x.float().view(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    s = (g.abs().amax(-1) / FP8_MAX).clamp_min(1e-12)
    return (g / s[..., None]).to(E4M3).view(x.shape), s


def _weights(E, N, K, tiled, gen):
    """N(0, 0.02) weights [E, N, K] with a scale for each 128 x 128 block, row-major or tile-first bytes."""
    nb, kb = N // BLOCK, K // BLOCK
    q = torch.empty((E, nb, kb, BLOCK, BLOCK) if tiled else (E, N, K), dtype=E4M3, device="cuda")
    s = torch.empty((E, nb, kb), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (N * K))
    for e in range(0, E, step):
        n = min(step, E - e)
        w = torch.randn((n, nb, kb, BLOCK, BLOCK), generator=gen, device="cuda", dtype=torch.bfloat16).float() * 0.02
        s[e:e + n] = (w.abs().amax((-1, -2)) / FP8_MAX).clamp_min(1e-12)
        t = (w / s[e:e + n, ..., None, None]).to(E4M3)
        q[e:e + n] = t if tiled else t.permute(0, 1, 3, 2, 4).reshape(n, N, K)
    return q, s


def _plan(ids, begin, count):
    """The dispatch plan of ids [T, k]: rows sorted by expert, then by place in ids."""
    T, k = ids.shape
    flat = ids.reshape(-1)
    local = (flat >= begin) & (flat < begin + count)
    key = torch.where(local, flat - begin, torch.full_like(flat, count))
    sorted_key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(sorted_key, torch.arange(count + 1, device=ids.device, dtype=key.dtype)).to(torch.int32)
    at = torch.arange(T * k, device=ids.device)
    row_token = torch.where(at < offsets[-1], order // k, torch.full_like(order, -1)).to(torch.int32)
    rows = torch.empty_like(order)
    rows[order] = at
    slot_row = torch.where(local, rows, torch.full_like(rows, -1)).view(T, k).to(torch.int32)
    return offsets, row_token, slot_row


def _routing(T, E, k, skew, gen):
    logits = torch.randn((T, E), generator=gen, device="cuda") + skew * torch.randn((E,), generator=gen, device="cuda")
    val, ids = torch.topk(logits, k, dim=1)
    return torch.softmax(val, 1), ids.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, op, k = case["T"], case["op"], case["k"]
    st = {"case": case}
    if op == "route":
        x = torch.randn((T, case["E"]), generator=gen, device="cuda") * 1.5
        if case["masked"]:
            x[torch.rand((T,), generator=gen, device="cuda") < case["masked"]] = -math.inf
        st["logits"] = x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        return st
    H = case["H"]
    if op == "block":
        bf = torch.bfloat16
        rows = max(1, k) * T
        st["y"] = torch.randn((rows, H), generator=gen, device="cuda", dtype=bf) * 0.5
        st["residual"] = torch.randn((T, H), generator=gen, device="cuda").to(torch.float32 if case["wide"] else bf)
        st["pre"] = (1 + 0.1 * torch.randn((H,), generator=gen, device="cuda")).to(bf)
        st["post"] = (1 + 0.1 * torch.randn((H,), generator=gen, device="cuda")).to(bf) if case["post"] else None
        shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[case["gate"]]
        st["gate"] = None if shape is None else torch.sigmoid(torch.randn(shape, generator=gen, device="cuda")).to(bf)
        if k:
            w, ids = _routing(T, 64, k, 0.5, gen)
            st["plan"] = (w, ids, *_plan(ids, 0, 64))
        return st
    E, I = case["E"], case["I"]
    w, ids = _routing(T, E, k, case["skew"], gen)
    st["plan"] = (w, ids, *_plan(ids, 0, E))
    st["most"] = int(torch.bincount(ids.reshape(-1).long(), minlength=E).max())  # rows of the busiest expert
    N, K = (2 * I, H) if op == "gate_up" else (H, I)
    st["W"], st["Ws"] = _weights(E, N, K, case["tiled"], gen)
    x = torch.randn((T if op == "gate_up" else T * k, K), generator=gen, device="cuda", dtype=torch.bfloat16)
    x[:: 101] *= 8  # a few tokens far above the others
    st["A"], st["As"] = _quant_rows(x)
    return st


# ------------------------------------------------------------------ the plain forms
def _plain_route(st):
    c = st["case"]
    x = st["logits"].float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    val, idx = torch.sort(x, dim=1, descending=True, stable=True)
    top, m = val[:, : c["k"]], val[:, :1]
    some = top > -math.inf
    ids = torch.where(some, idx[:, : c["k"]], torch.full_like(idx[:, : c["k"]], -1)).to(torch.int32)
    e = torch.where(some, torch.where(top == m, torch.ones_like(top), torch.exp(top - m)), torch.zeros_like(top))
    if c["renormalize"]:
        total = e.sum(1, keepdim=True)
    else:
        total = torch.where(val == m, torch.ones_like(val), torch.exp(val - m)).sum(1, keepdim=True)
    weights = torch.where(some, e / total, torch.zeros_like(e))
    offsets, row_token, slot_row = _plan(ids, c["begin"], c["count"])
    return {"weights": weights, "ids": ids, "offsets": offsets, "row_token": row_token, "slot_row": slot_row}


def _wide_weights(q, s):
    """[n, N, K] fp32 of e4m3 weights in either layout and their block scales."""
    n, nb, kb = s.shape
    if q.dim() == 5:
        w = (q.float() * s[..., None, None]).permute(0, 1, 3, 2, 4)
    else:
        w = q.float().view(n, nb, BLOCK, kb, BLOCK) * s[:, :, None, :, None]
    return w.reshape(n, nb * BLOCK, kb * BLOCK)


def _plain_grouped(st, x):
    """x [R, K] fp32 in row order times each row's expert: [R, N] fp32."""
    offsets = st["plan"][2]
    E, R, most = st["W"].shape[0], x.shape[0], st["most"]
    at = torch.arange(R, device=x.device)
    expert = torch.searchsorted(offsets[1:].long(), at, right=True)
    if R <= E:  # only the weights that are asked for
        return torch.bmm(_wide_weights(st["W"][expert], st["Ws"][expert]), x[:, :, None])[:, :, 0]
    place = at - offsets.long()[expert]
    pad = torch.zeros((E, most, x.shape[1]), dtype=torch.float32, device=x.device)
    pad[expert, place] = x
    return torch.bmm(pad, _wide_weights(st["W"], st["Ws"]).transpose(1, 2))[expert, place]


def _plain_gate_up(st):
    A, As, row_token = st["A"], st["As"], st["plan"][3].long()
    x = (A.float().view(A.shape[0], -1, BLOCK) * As[..., None]).view(A.shape)[row_token]
    c = _plain_grouped(st, x)
    I = c.shape[1] // 2
    g, u = c[:, :I], c[:, I:]
    y = (g / (1 + torch.exp(-g)) * u).view(c.shape[0], I // BLOCK, BLOCK)
    s = y.abs().amax(-1).clamp_min(1e-10) / FP8_MAX
    q = (y * (1 / s)[..., None]).clamp(-FP8_MAX, FP8_MAX).to(E4M3)
    return {"Q": q.view(c.shape[0], I), "Qs": s}


def _plain_down(st):
    A, As = st["A"], st["As"]
    x = (A.float().view(A.shape[0], -1, BLOCK) * As[..., None]).view(A.shape)
    return _plain_grouped(st, x).to(torch.bfloat16)


SCALE, RESIDUAL_SCALE, EPS = 0.75, 0.9, 1e-6


def _plain_block(st):
    y = st["y"].float()
    if "plan" in st:
        w, slot_row = st["plan"][0], st["plan"][4].long()
        z = (y[slot_row] * w[..., None]).sum(1)
    else:
        z = y
    if st["post"] is not None:
        z = z * torch.rsqrt((z * z).mean(1, keepdim=True) + EPS) * st["post"].float()
    if st["gate"] is not None:
        z = z * st["gate"].float()
    h = RESIDUAL_SCALE * st["residual"].float() + SCALE * z
    v = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * st["pre"].float()
    q, s = _quant_rows(v)
    return {"residual": h.to(st["residual"].dtype), "A": q, "As": s}


# ------------------------------------------------------------------ one pass
def _package():
    at = str(Path(__file__).resolve().parents[1] / "ucloud-ai-infra_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from fp8_hand_b200 import ops
    return ops


def _own_run(st):
    ops, c = _package(), st["case"]
    if c["op"] == "route":
        r = ops.moe_route(st["logits"], c["k"], renormalize=c["renormalize"], experts=(c["begin"], c["count"]))
        return {"weights": r.weights, "ids": r.ids, "offsets": r.offsets, "row_token": r.row_token, "slot_row": r.slot_row}
    route = ops.MoeRoute(*st["plan"]) if "plan" in st else None
    if c["op"] == "gate_up":
        q, s = ops.grouped_gemm_silu_quant(st["A"], st["W"], st["As"], st["Ws"], route, b_tiled=c["tiled"])
        return {"Q": q, "Qs": s}
    if c["op"] == "down":
        return ops.grouped_gemm(st["A"], st["W"], st["As"], st["Ws"], route, b_tiled=c["tiled"])
    h, a, s = ops.block_norm_quant(st["y"], st["residual"], post_weight=st["post"], gate=st["gate"], scale=SCALE,
                                   residual_scale=RESIDUAL_SCALE, pre_weight=st["pre"], eps=EPS, route=route)
    return {"residual": h, "A": a, "As": s}


def run(state):
    if own:
        return _own_run(state)
    return {"route": _plain_route, "gate_up": _plain_gate_up, "down": _plain_down,
            "block": _plain_block}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits
def _e4m3_64(v):
    """The e4m3 value nearest to v, ties to even, as float64."""
    a = v.abs().clamp(max=FP8_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(v) * torch.round(a / step) * step


def _exact_rows(st, e, rows):
    """float64 products of the rows `rows` [n, K] with expert e's weights, block by block."""
    q, s = st["W"][e], st["Ws"][e].double()
    if q.dim() == 4:
        q = q.permute(0, 2, 1, 3).reshape(q.shape[0] * BLOCK, -1)
    w = q.double() * s.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
    return rows @ w.T


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "route":
        x = st["logits"].double()
        order = torch.argsort(-x, dim=1, stable=True)[:, : case["k"]]
        top = torch.gather(x, 1, order)
        base = x.amax(1, keepdim=True)
        of = top if case["renormalize"] else x
        w = torch.exp(top - base) / torch.exp(of - base).sum(1, keepdim=True)
        return {"weights": torch.nan_to_num(w, nan=0.0), "ids": None, "offsets": None, "row_token": None, "slot_row": None}
    if op == "block":
        y, h = st["y"].double(), st["residual"].double()
        if "plan" in st:
            z = torch.zeros_like(h)
            for s in range(case["k"]):
                z += st["plan"][0][:, s:s + 1].double() * y[st["plan"][4][:, s].long()]
        else:
            z = y
        if st["post"] is not None:
            z = z / ((z ** 2).mean(1, keepdim=True) + EPS).sqrt() * st["post"].double()
        if st["gate"] is not None:
            z = z * st["gate"].double()
        h = RESIDUAL_SCALE * h + SCALE * z
        v = h / ((h ** 2).mean(1, keepdim=True) + EPS).sqrt() * st["pre"].double()
        g = v.view(v.shape[0], -1, BLOCK)
        s = (g.abs().amax(-1) / FP8_MAX).clamp_min(1e-12)
        return {"residual": h, "A": _e4m3_64(g / s[..., None]).view(v.shape), "As": s}
    offsets, tokens = st["plan"][2].tolist(), st["plan"][3].long()
    A = st["A"].double() * st["As"].double().repeat_interleave(BLOCK, 1)
    out = []
    for e in range(case["E"]):
        lo, hi = offsets[e], offsets[e + 1]
        if hi > lo:
            out.append(_exact_rows(st, e, A[tokens[lo:hi]] if op == "gate_up" else A[lo:hi]))
    c = torch.cat(out)
    if op == "down":
        return c
    g, u = c.chunk(2, 1)
    y = (g * torch.sigmoid(g) * u).view(c.shape[0], -1, BLOCK)
    s = y.abs().amax(-1).clamp_min(1e-10) / FP8_MAX
    return {"Q": _e4m3_64(y / s[..., None]).view(c.shape[0], -1), "Qs": s}
