"""64-bit CPU oracle of the mixture-of-experts operators. TEST INFRASTRUCTURE ONLY (see oracle.py).

Plain restatements of the formulas in float64 with loops over experts and tokens, and the error bounds that fp32
arithmetic of the same formulas may have. The reference has no mixture of experts; the grouped products repeat its dense
per-128-block formulas (oracle.py) for each expert.
"""
from __future__ import annotations

import math

import torch

BLOCK = 128
FP8_MAX = 448.0
U = 2.0 ** -24  # half an ulp of fp32, relative


# ----------------------------------------------------------------------------- router
def route(logits: torch.Tensor, k: int, renormalize: bool = True, scale: float = 1.0):
    """(ids int32 [T, k], weights float64 [T, k])."""
    T, E = logits.shape
    ids = torch.full((T, k), -1, dtype=torch.int32)
    w = torch.zeros((T, k), dtype=torch.float64)
    for t in range(T):
        x = [float(v) for v in logits[t].float()]
        live = [e for e in range(E) if not math.isnan(x[e]) and x[e] > -math.inf]
        if not live:
            continue
        top = sorted(live, key=lambda e: (-x[e], e))[:k]
        m = max(x[e] for e in live)
        p = {e: 1.0 if x[e] == m else math.exp(x[e] - m) for e in live}
        total = sum(p[e] for e in (top if renormalize else live))
        for s, e in enumerate(top):
            ids[t, s], w[t, s] = e, scale * p[e] / total
    return ids, w


def plan(ids: torch.Tensor, begin: int, count: int):
    """(offsets, row_token, slot_row) of ids [T, k] for the local experts [begin, begin + count)."""
    T, k = ids.shape
    slot_row = torch.full((T, k), -1, dtype=torch.int32)
    row_token = torch.full((T * k,), -1, dtype=torch.int32)
    offsets, r = [0], 0
    flat = ids.reshape(-1).tolist()
    for e in range(begin, begin + count):
        for i, v in enumerate(flat):
            if v == e:
                row_token[r] = i // k
                slot_row[i // k, i % k] = r
                r += 1
        offsets.append(r)
    return torch.tensor(offsets, dtype=torch.int32), row_token, slot_row


# ----------------------------------------------------------------------------- grouped products
def wide(q: torch.Tensor, s: torch.Tensor, rows: int) -> torch.Tensor:
    return q.double() * s.double().repeat_interleave(rows, 0).repeat_interleave(BLOCK, 1)


def grouped(A, As, B, Bs, offsets, sources):
    """Products of rows `sources` of A with their expert's weights: (float64 [n, N], the bound on fp32's error),
    n = offsets[-1]. The bound: each K block's 128 products are summed with at most one ulp (2U) an addition,
    the scale product and the fma round once each, and KB blocks are added."""
    KB = A.shape[1] // BLOCK
    c, tol = [], []
    for e in range(B.shape[0]):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if hi == lo:
            continue
        a, w = wide(A, As, 1)[sources[lo:hi].long()], wide(B[e], Bs[e], BLOCK)
        c.append(a @ w.T)
        tol.append((2 * BLOCK + KB + 3) * U * (a.abs() @ w.abs().T))
    if not c:
        z = torch.zeros((0, B.shape[1]), dtype=torch.float64)
        return z, z
    return torch.cat(c), torch.cat(tol)


def silu_mul(c: torch.Tensor, tol: torch.Tensor):
    """y = silu(g) * u of [g | u] and the bound on its fp32 error: |silu'| <= 1.1; the exponential's argument
    scales its error, so an exp and a divide of a few ulp come to (8 + 2 |g|) ulp of y."""
    inter = c.shape[1] // 2
    g, u, tg, tu = c[:, :inter], c[:, inter:], tol[:, :inter], tol[:, inter:]
    s = g * torch.sigmoid(g)
    y = s * u
    return y, 1.1 * u.abs() * tg + s.abs() * tu + 1.1 * tg * tu + (8 + 2 * g.abs()) * 2 * U * y.abs()


def check_quant(q: torch.Tensor, s: torch.Tensor, v: torch.Tensor, tol: torch.Tensor, floor: float):
    """An e4m3 group quant (q, s) of values v that are known within tol: the scale is max(amax / 448, floor) within
    the amax's error and two roundings, and q * s is within half an e4m3 step of v (2^-4 relative, 2^-10 of the
    scale below the normals; the smallest normal is 2^-6), plus tol and the arithmetic's own four roundings."""
    n = v.shape[-1] // BLOCK
    g, tg = v.view(-1, n, BLOCK), tol.view(-1, n, BLOCK)
    ref = (g.abs().amax(-1) / FP8_MAX).clamp_min(floor)
    err = (s.double().view(-1, n) - ref).abs()
    assert bool((err <= tg.amax(-1) / FP8_MAX + 4 * U * ref).all()), (err / ref).max()
    sd = s.double().view(-1, n, 1)
    back = q.float().double().view(-1, n, BLOCK) * sd
    lim = (2.0 ** -4 + 8 * U) * g.abs() + 2.0 ** -10 * sd + 1.0625 * tg + tg.amax(-1, keepdim=True)
    assert bool(((back - g).abs() <= lim).all()), ((back - g).abs() / lim).max()


# ----------------------------------------------------------------------------- the block's end
def block(y, residual, *, post=None, gate=None, scale=1.0, residual_scale=1.0, pre=None, eps=1e-6, weights=None,
          slot_row=None):
    """(h, its fp32 error bound, v or None, its bound). Bounds: a sum of n terms (n + 1) U of the absolute sum; the
    sum of squares over H, kept in a chain of at most 32 per thread, a butterfly of 5 and at most 16 warp totals:
    56 U relative, half of it in 1/sqrt, plus the relative error of the terms, and three roundings."""
    T, H = residual.shape
    yd = y.double()
    if weights is not None:
        z = torch.zeros((T, H), dtype=torch.float64)
        mag = torch.zeros_like(z)
        for t in range(T):
            for s in range(weights.shape[1]):
                r = int(slot_row[t, s])
                if r >= 0:
                    z[t] += float(weights[t, s]) * yd[r]
                    mag[t] += (float(weights[t, s]) * yd[r]).abs()
        tol = (weights.shape[1] + 1) * U * mag
    else:
        z, tol = yd, torch.zeros((T, H), dtype=torch.float64)

    def norm(x, tx, w):
        ms = (x ** 2).mean(1, keepdim=True) + eps
        # relative error of the mean square: the terms' (2 |x| tx summed) and the summation's
        rel = (2 * (x.abs() * tx).mean(1, keepdim=True) + (tx ** 2).mean(1, keepdim=True)) / ms + 58 * U
        rs = ms.rsqrt()
        wd = w.double()
        v = x * rs * wd
        return v, rs * wd.abs() * tx * (1 + rel) + v.abs() * (rel / 2 * (1 + rel) + 6 * U)

    if post is not None:
        z, tol = norm(z, tol, post)
    b = scale if gate is None else scale * gate.double()
    a = residual_scale * residual.double()
    h = a + b * z
    tol = (b.abs() if torch.is_tensor(b) else abs(b)) * tol + 4 * U * (a.abs() + (b * z).abs())
    if pre is None:
        return h, tol, None, None
    v, tv = norm(h, tol, pre)
    return h, tol, v, tv
