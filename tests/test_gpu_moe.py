"""The mixture-of-experts operators on the GPU against the 64-bit oracle, whose error bounds follow from the formulas
(oracle/moe.py): plans and ids exact, products and norms within the bound of fp32 arithmetic plus the output's rounding."""
import math

import pytest
import torch

from oracle import moe as M
from oracle import oracle as O

pytestmark = pytest.mark.gpu

BF16_HALF = 2.0 ** -8 * 1.01  # half an ulp of a bf16 (8-bit significand), and the error's own rounding


def _ops():
    from fp8_hand_b200 import ops
    return ops


def _within(x, ref, tol, half=0.0):
    """|x - ref| <= tol + half * |value| + the smallest step of the output's type."""
    x = x.cpu().double()
    err, lim = (x - ref).abs(), tol + half * (ref.abs() + tol) + 1e-37
    assert bool((err <= lim).all()), float((err / lim).max())


# ----------------------------------------------------------------------------- router
def _check_plan(r, ids, begin, count):
    off, row_token, slot_row = M.plan(ids, begin, count)
    assert torch.equal(r.offsets.cpu(), off)
    assert torch.equal(r.row_token.cpu(), row_token)
    assert torch.equal(r.slot_row.cpu(), slot_row)


def _check_route(r, logits, k, renormalize=True, scale=1.0, begin=0, count=None):
    T, E = logits.shape
    ids, w = M.route(logits, k, renormalize, scale)
    assert torch.equal(r.ids.cpu(), ids)
    # exp of at most 2 ulp, a sum of at most E terms, divide, scale
    _within(r.weights, w, torch.full_like(w, 0.0), half=(2 * (4 + math.ceil(E / 32) + 5) + 4) * M.U)
    _check_plan(r, ids, begin, E if count is None else count)


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (31, 33, 4), (32, 8, 8), (33, 160, 6), (65, 257, 3), (777, 128, 8),
                                   (130, 512, 32), (4800, 16, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_route(cuda_lib, T, E, k, dtype):
    g = torch.Generator().manual_seed(T * E + k)
    logits = (torch.randn(T, E, generator=g) * 3).to(dtype)
    logits[T // 2] = (logits[T // 2] * 2).round() / 2  # ties
    _check_route(_ops().moe_route(logits.cuda(), k), logits, k)


def test_route_ties_and_zeros(cuda_lib):
    logits = torch.zeros(40, 96)
    logits[:, 1::2] = -0.0
    logits[20:] = torch.randint(-1, 2, (20, 96), generator=torch.Generator().manual_seed(1)).float()
    _check_route(_ops().moe_route(logits.cuda(), 7, scale=2.5), logits, 7, scale=2.5)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_masked(cuda_lib, renormalize):
    """-inf, NaN, +inf, the type's lowest value, and rows that the mask leaves nothing or too little of."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(70, 48, generator=g)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 3:] = -math.inf                              # three candidates for five slots
    x[3, ::2] = math.nan
    x[4, 7], x[4, 9] = math.inf, math.inf
    x[5] = torch.finfo(torch.float32).min
    x[6, 1:] = torch.finfo(torch.float32).min
    x[7, :] = -math.inf
    x[7, 47] = torch.finfo(torch.float32).min
    x[8, 0] = torch.finfo(torch.float32).max
    x[69] = -math.inf
    _check_route(_ops().moe_route(x.cuda(), 5, renormalize=renormalize), x, 5, renormalize)


def test_route_strided_and_local(cuda_lib):
    g = torch.Generator().manual_seed(3)
    big = torch.randn(300, 131, generator=g).to(torch.bfloat16)
    x = big[:, 1:100]                                  # odd stride, odd start
    for begin, count in ((0, 99), (50, 49), (98, 1)):
        r = _ops().moe_route(big.cuda()[:, 1:100], 6, renormalize=False, experts=(begin, count))
        _check_route(r, x, 6, False, 1.0, begin, count)
    t = torch.randn(20, 77, generator=g)
    _check_route(_ops().moe_route(t.cuda().t(), 4), t.t(), 4)
    _check_route(_ops().moe_route(t[:1].cuda().expand(50, 77), 4), t[:1].expand(50, 77), 4)


def test_route_empty(cuda_lib):
    r = _ops().moe_route(torch.zeros(0, 16, device="cuda"), 2)
    assert r.weights.shape == (0, 2) and r.row_token.numel() == 0 and r.offsets.tolist() == [0] * 17


@pytest.mark.parametrize("T,k,E,begin,count", [(1, 1, 4, 0, 4), (50, 8, 40, 0, 40), (700, 5, 300, 100, 150), (6000, 3, 512, 0, 512)])
def test_dispatch(cuda_lib, T, k, E, begin, count):
    """Given ids: -1 and ids of other ranks have no row, an expert may fill several slots of a token."""
    ids = torch.randint(-1, E, (T, k), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    ids[T // 2] = ids[T // 2, 0]
    r = _ops().moe_dispatch(ids.cuda(), None, E, experts=(begin, count))
    _check_plan(r, ids, begin, count)
    r = _ops().moe_dispatch(torch.full_like(ids, -1).cuda(), None, E)
    assert int(r.offsets.abs().max()) == 0 and bool((r.slot_row == -1).all()) and bool((r.row_token == -1).all())


@pytest.mark.parametrize("T,E,k", [(29, 64, 9), (64, 16, 10), (200, 160, 32), (512, 40, 9), (513, 64, 9), (700, 512, 32),
                                   (9500, 24, 5), (20000, 16, 8)])
def test_plan_several_batches(cuda_lib, T, E, k):
    """CTAs that rank their pairs in several batches: more than 256 pairs each, in one cluster (up to 512 tokens) and in two
    launches. Few experts in a token's reach make long runs of one expert across batches; every call gives the same plan."""
    g = torch.Generator().manual_seed(T + E + k)
    logits = torch.randn(T, E, generator=g) + 2 * torch.randn(E, generator=g)
    r = _ops().moe_route(logits.cuda(), k)
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
    assert torch.equal(r.ids.cpu(), ids)
    _check_plan(r, ids, 0, E)
    begin, count = E // 4, E // 2
    for _ in range(10):
        _check_same(_ops().moe_route(logits.cuda(), k), r)
        _check_same(_ops().moe_dispatch(r.ids, None, E), r)
    _check_plan(_ops().moe_dispatch(r.ids, None, E, experts=(begin, count)), ids, begin, count)


def _check_same(r, want):
    for name in ("offsets", "row_token", "slot_row"):
        assert torch.equal(getattr(r, name), getattr(want, name)), name


# ----------------------------------------------------------------------------- grouped products
def _case(counts, N, K, seed, spread=0):
    """Rows per expert -> (route tensors, weights and scales, tokens): every token in one slot, in shuffled order."""
    g = torch.Generator().manual_seed(seed)
    E, R = len(counts), sum(counts)
    ids = torch.cat([torch.full((c,), e, dtype=torch.int32) for e, c in enumerate(counts)])
    ids = torch.cat([ids, torch.full((spread,), -1, dtype=torch.int32)])
    ids = ids[torch.randperm(R + spread, generator=g)][:, None].contiguous()
    q, s = zip(*[O.make_weight(N, K, seed + 10 + e) for e in range(E)])
    x = O.make_activation(R + spread, K, seed + 1, outlier_frac=0.05)
    A, As = O.group_quant(x)
    return ids, torch.stack([t.view(torch.uint8) for t in q]).view(torch.float8_e4m3fn), torch.stack(s), A, As


def _route_for(ids, E, mean):
    """The plan, with a number of experts that makes the expected rows per expert `mean` (it picks the kernel)."""
    r = _ops().moe_dispatch(ids.cuda(), None, E)
    if mean:
        r.num_experts = max(E, ids.numel() // mean)
    return r


def _tiles(B):
    E, N, K = B.shape
    return _ops().pack_tiles(B.reshape(E * N, K).cuda()).view(E, N // 128, K // 128, 128, 128)


COUNTS = {"one": [0, 1, 0], "few": [3, 0, 1, 16, 17, 0, 2], "edges": [15, 16, 17, 31, 33, 0, 63, 64, 65],
          "many": [127, 128, 0, 129, 300], "single": [0, 0, 400], "none": [0, 0]}


@pytest.mark.parametrize("counts", sorted(COUNTS))
@pytest.mark.parametrize("mean", [1, 10, 20, 50, 0])
@pytest.mark.parametrize("N,K,tiled", [(128, 128, False), (384, 640, True), (640, 1152, False)])
def test_grouped_gemm(cuda_lib, counts, mean, N, K, tiled):
    """Every kernel variant (mean rows per expert) at row counts around its tiles, rows of no expert in between, an
    odd number of weight blocks, one K block; both outputs, both ways to read the rows. Rows past the last
    expert's are not written."""
    ops = _ops()
    ids, B, Bs, A, As = _case(COUNTS[counts], N, K, 7, spread=9)
    r = _route_for(ids, len(COUNTS[counts]), mean)
    n = sum(COUNTS[counts])
    off, src, _ = M.plan(ids, 0, len(COUNTS[counts]))
    W = _tiles(B) if tiled else B.cuda()
    ref, tol = M.grouped(A, As, B, Bs, off, src)
    out = torch.full((ids.numel(), N), 7.0, device="cuda")
    ops.grouped_gemm(A.cuda(), W, As.cuda(), Bs.cuda(), r, b_tiled=tiled, gather=True, out=out)
    _within(out[:n], ref, tol)
    assert bool((out[n:] == 7.0).all())
    rows = torch.cat([src[:n].long(), torch.zeros(9, dtype=torch.long)])  # the same rows laid out in row order
    wide = torch.full((ids.numel(), N + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.grouped_gemm(A.view(torch.uint8)[rows].view(torch.float8_e4m3fn).cuda(), W, As[rows].cuda(), Bs.cuda(), r,
                     b_tiled=tiled, out=wide[:, :N])
    _within(wide[:n, :N], ref, tol, BF16_HALF)
    assert bool((wide[n:] == 7.0).all()) and bool((wide[:, N:] == 7.0).all())
    from fp8_hand_b200 import _native
    assert _native.status() == 0


@pytest.mark.parametrize("counts", sorted(COUNTS))
@pytest.mark.parametrize("mean", [1, 10, 20, 50, 0])
@pytest.mark.parametrize("inter,K,tiled", [(128, 128, True), (384, 640, False)])
def test_grouped_gemm_silu_quant(cuda_lib, counts, mean, inter, K, tiled):
    ops = _ops()
    ids, B, Bs, A, As = _case(COUNTS[counts], 2 * inter, K, 11, spread=5)
    r = _route_for(ids, len(COUNTS[counts]), mean)
    n = sum(COUNTS[counts])
    off, src, _ = M.plan(ids, 0, len(COUNTS[counts]))
    y, tol = M.silu_mul(*M.grouped(A, As, B, Bs, off, src))
    Q, Qs = ops.grouped_gemm_silu_quant(A.cuda(), _tiles(B) if tiled else B.cuda(), As.cuda(), Bs.cuda(), r, b_tiled=tiled)
    if n:
        M.check_quant(Q[:n].cpu(), Qs[:n].cpu(), y, tol, 1e-10 / 448)
    from fp8_hand_b200 import _native
    assert _native.status() == 0


@pytest.mark.parametrize("T", [1, 7, 300])
def test_grouped_several_slots(cuda_lib, T):
    """Tokens with several slots: one token's row is read by several experts; zero and huge tokens among them."""
    ops = _ops()
    E, k, K, inter = 6, 3, 512, 256
    g = torch.Generator().manual_seed(T)
    logits = torch.randn(T, E, generator=g)
    x = O.make_activation(T, K, 5)
    x[0] = 0
    x[T // 2] *= 1000
    A, As = O.group_quant(x)
    ws = [O.make_weight(2 * inter, K, 30 + e) for e in range(E)]
    B, Bs = torch.stack([w.view(torch.uint8) for w, _ in ws]).view(torch.float8_e4m3fn), torch.stack([s for _, s in ws])
    r = ops.moe_route(logits.cuda(), k)
    off, src, _ = M.plan(r.ids.cpu(), 0, E)
    y, tol = M.silu_mul(*M.grouped(A, As, B, Bs, off, src))
    Q, Qs = ops.grouped_gemm_silu_quant(A.cuda(), B.cuda(), As.cuda(), Bs.cuda(), r)
    M.check_quant(Q.cpu(), Qs.cpu(), y, tol, 1e-10 / 448)
    Q2, Qs2 = ops.grouped_gemm_silu_quant(A.cuda(), B.cuda(), As.cuda(), Bs.cuda(), r)
    assert torch.equal(Q.view(torch.uint8), Q2.view(torch.uint8)) and torch.equal(Qs, Qs2)


SPLIT_COUNTS = {"few": [3, 0, 1, 16, 17, 0, 2], "many": [100, 0, 300, 3]}


def _plan_is(rows, E, N, K, fused, want):
    from fp8_hand_b200 import _native
    assert _native.num_sms() == 148, "the clusters below are chosen for 148 SMs"
    p = _native.grouped_plan(rows, E, N, K, fused)
    assert (p["kind"], p["tile_rows"], p["cluster"]) == (1, *want), p


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("counts", sorted(SPLIT_COUNTS))
@pytest.mark.parametrize("tile", [16, 32])
@pytest.mark.parametrize("K,cluster", [(2048, 2), (2176, 2), (4096, 4), (5248, 4), (8192, 8), (8320, 8)])
def test_grouped_clusters(cuda_lib, fused, counts, tile, K, cluster):
    """Tiles whose K is split over 2, 4 and 8 CTAs, evenly and not: tiles with fewer rows than CTAs (some finish no row), and
    more tiles than clusters, so that each uses its exchange buffer several times. Every run gives the same bits."""
    ops = _ops()
    c = SPLIT_COUNTS[counts]
    E, N = len(c), 512 if fused else 256
    ids, B, Bs, A, As = _case(c, N, K, 23)
    R = ids.numel()
    rows = {16: E, 32: 5 * E}[tile]                    # rows that the call expects, by the experts in all
    experts = R * E // rows if counts == "many" else {16: R, 32: E}[tile]
    rows = min(R, -(-R * E // experts))
    _plan_is(rows, E, N, K, fused, (tile, cluster))
    r = ops.moe_dispatch(ids.cuda(), None, E)
    r.num_experts = experts
    off, src, _ = M.plan(ids, 0, E)
    ref, tol = M.grouped(A, As, B, Bs, off, src)
    dev = [t.cuda() for t in (A, B, As, Bs)]
    if fused:
        y, ty = M.silu_mul(ref, tol)
        Q, Qs = ops.grouped_gemm_silu_quant(*dev, r)
        M.check_quant(Q.cpu(), Qs.cpu(), y, ty, 1e-10 / 448)
        for _ in range(5):
            Q2, Qs2 = ops.grouped_gemm_silu_quant(*dev, r)
            assert torch.equal(Q.view(torch.uint8), Q2.view(torch.uint8)) and torch.equal(Qs, Qs2)
    else:
        out = ops.grouped_gemm(*dev, r, gather=True, out_dtype=torch.float32)
        _within(out, ref, tol)
        order = src.long()
        rows_in_order = A.view(torch.uint8)[order].view(torch.float8_e4m3fn).cuda()
        tiles = _tiles(B)
        for _ in range(5):
            assert torch.equal(ops.grouped_gemm(*dev, r, gather=True, out_dtype=torch.float32), out)
            got = ops.grouped_gemm(rows_in_order, tiles, As[order].cuda(), dev[3], r, b_tiled=True)
            assert torch.equal(got, out.to(torch.bfloat16))
    from fp8_hand_b200 import _native
    assert _native.status() == 0


@pytest.mark.parametrize("tile", [16, 32])
def test_grouped_clusters_more_tiles_than_sms(cuda_lib, tile):
    """The fused product on two CTAs per tile with more tiles than SMs: every cluster walks several tiles."""
    ops = _ops()
    E, N, K = 38, 1024, 2048
    c = [1 + e % 3 for e in range(E)]
    c[5], c[20] = 40, 17
    ids, B, Bs, A, As = _case(c, N, K, 29)
    R = ids.numel()
    assert E < R <= 4 * E
    _plan_is(R, E, N, K, True, (16, 2))
    r = ops.moe_dispatch(ids.cuda(), None, E)
    if tile == 32:  # the same rows, and slots of no expert
        spread = 4 * E + 1 - R
        ids = torch.cat([ids, torch.full((spread, 1), -1, dtype=torch.int32)])
        A = torch.cat([A.view(torch.uint8), torch.zeros(spread, K, dtype=torch.uint8)]).view(torch.float8_e4m3fn)
        As = torch.cat([As, torch.ones(spread, K // 128)])
        _plan_is(ids.numel(), E, N, K, True, (32, 2))
        r = ops.moe_dispatch(ids.cuda(), None, E)
    off, src, _ = M.plan(ids, 0, E)
    y, tol = M.silu_mul(*M.grouped(A, As, B, Bs, off, src))
    dev = [t.cuda() for t in (A, _tiles(B), As, Bs)]
    Q, Qs = ops.grouped_gemm_silu_quant(*dev, r, b_tiled=True)
    M.check_quant(Q[:R].cpu(), Qs[:R].cpu(), y, tol, 1e-10 / 448)
    for _ in range(10):
        Q2, Qs2 = ops.grouped_gemm_silu_quant(*dev, r, b_tiled=True)
        assert torch.equal(Q[:R].view(torch.uint8), Q2[:R].view(torch.uint8)) and torch.equal(Qs[:R], Qs2[:R])
    from fp8_hand_b200 import _native
    assert _native.status() == 0


@pytest.mark.parametrize("mean", [1, 10, 50])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_silu_quant_not_finite(cuda_lib, mean, bad):
    """A column that is NaN (an e4m3 NaN in a gate row of the weights) stays one NaN: its group's scale comes from the other
    127 columns, in every kernel. Groups of infinite columns have an infinite scale."""
    ops = _ops()
    counts, inter = [60, 0, 7], 384  # by mean: token tiles of 16 and 32 rows, row tiles
    ids, B, Bs, A, As = _case(counts, 2 * inter, 256, 19)
    off, src, _ = M.plan(ids, 0, 3)
    y, tol = M.silu_mul(*M.grouped(A, As, B, Bs, off, src))
    cols = [5, 130, 131, 383]
    if bad == "nan":
        for c in cols:
            B.view(torch.uint8)[0, c, 40] = 0x7F
    else:
        Bs = Bs.clone()
        Bs[0, 0] = math.inf  # the gates of the first 128 columns: infinite, or NaN where an infinite sum has both signs
    Q, Qs = ops.grouped_gemm_silu_quant(A.cuda(), B.cuda(), As.cuda(), Bs.cuda(), _route_for(ids, 3, mean))
    Q, Qs, n = Q.cpu(), Qs.cpu(), counts[0]
    if bad == "nan":
        assert bool(Q.float()[:n, cols].isnan().all())
        Q.view(torch.uint8)[:n, cols] = 0
        y[:n, cols] = tol[:n, cols] = 0
        M.check_quant(Q, Qs, y, tol, 1e-10 / 448)
    else:
        assert not bool(Q.float()[n:].isnan().any()) and not bool(Q.float()[:, 128:].isnan().any())
        M.check_quant(Q[n:], Qs[n:], y[n:], tol[n:], 1e-10 / 448)
        M.check_quant(Q[:n, 128:], Qs[:n, 1:], y[:n, 128:], tol[:n, 128:], 1e-10 / 448)


# ----------------------------------------------------------------------------- the block's end
def _block_case(T, H, k, wide, seed):
    g = torch.Generator().manual_seed(seed)
    bf = torch.bfloat16
    rows = T * max(1, k) + 3 if k else T
    y = torch.randn(rows, H, generator=g).to(bf)
    res = torch.randn(T, H, generator=g).to(torch.float32 if wide else bf)
    post = (1 + 0.2 * torch.randn(H, generator=g)).to(bf)
    pre = (1 + 0.2 * torch.randn(H, generator=g)).to(bf)
    w = slot = None
    if k:
        w = torch.rand(T, k, generator=g)
        slot = torch.randperm(T * k, generator=g).view(T, k).to(torch.int32)
        slot[torch.rand(T, k, generator=g) < 0.2] = -1
        slot[T // 2] = -1                              # a token with no row at all
    return y, res, post, pre, w, slot, g


def _route_of(w, slot):
    if w is None:
        return None
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    return _ops().MoeRoute(w.cuda(), slot.cuda(), e, e, slot.cuda())


def _check_block(got, want, wide, half=BF16_HALF):
    h, th, v, tv = want
    if v is None:
        _within(got, h, th, 2 * M.U if wide else half)
        return
    _within(got[0], h, th, 2 * M.U if wide else half)
    M.check_quant(got[1].cpu(), got[2].cpu(), v, tv, 1e-12)


@pytest.mark.parametrize("T,H,k,wide", [(1, 128, 0, False), (1, 5120, 8, False), (3, 2176, 1, True), (37, 5120, 6, False),
                                        (700, 640, 2, True), (5, 16384, 3, False), (2, 8192, 0, True)])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_block_norm(cuda_lib, T, H, k, wide, gate):
    y, res, post, pre, w, slot, g = _block_case(T, H, k, wide, T + H + k)
    shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[gate]
    gt = None if shape is None else torch.sigmoid(torch.randn(shape, generator=g)).to(torch.bfloat16)
    kw = dict(scale=0.7, residual_scale=1.3, eps=1e-5)
    dev = dict(post_weight=post.cuda(), gate=None if gt is None else gt.cuda(), route=_route_of(w, slot))
    want = M.block(y, res, post=post, gate=gt, pre=pre, weights=w, slot_row=slot, **kw)
    _check_block(_ops().block_norm_quant(y.cuda(), res.cuda(), pre_weight=pre.cuda(), **dev, **kw), want, wide)
    inplace = res.cuda()
    out = _ops().block_norm_quant(y.cuda(), inplace, out=inplace, **dev, **kw)
    assert out is inplace
    _check_block(out, (want[0], want[1], None, None), wide)


@pytest.mark.parametrize("T,H,k,wide", [(320, 2560, 4, False), (310, 2688, 1, True), (301, 5248, 8, False),
                                        (160, 7168, 5, True), (170, 10240, 0, False), (150, 10368, 2, True),
                                        (151, 16384, 8, True)])
def test_block_row_lengths(cuda_lib, T, H, k, wide):
    """The first and last lengths of the kernel's shapes, with several rows per CTA."""
    y, res, post, pre, w, slot, g = _block_case(T, H, k, wide, T + H + k)
    gt = torch.sigmoid(torch.randn(H, generator=g)).to(torch.bfloat16)
    kw = dict(scale=0.9, residual_scale=1.1, eps=1e-6)
    got = _ops().block_norm_quant(y.cuda(), res.cuda(), post_weight=post.cuda(), gate=gt.cuda(), pre_weight=pre.cuda(),
                                  route=_route_of(w, slot), **kw)
    _check_block(got, M.block(y, res, post=post, gate=gt, pre=pre, weights=w, slot_row=slot, **kw), wide)


@pytest.mark.parametrize("T,H", [(14300, 128), (2300, 1024), (2300, 1152), (2300, 2560), (1350, 2688), (1000, 5120),
                                 (460, 5248), (460, 10240), (460, 10368), (460, 16384)])
@pytest.mark.parametrize("k,wide", [(0, False), (6, False), (5, True)])
def test_block_many_rows_per_cta(cuda_lib, T, H, k, wide):
    """The first and the last length of each of the kernel's shapes with at least three rows per CTA: the ring's stages, both
    residual slots and both sets of sums are used again."""
    y, res, post, pre, w, slot, g = _block_case(T, H, k, wide, T + H + k)
    gt = torch.sigmoid(torch.randn(T, 1, generator=g)).to(torch.bfloat16)
    kw = dict(scale=0.8, residual_scale=0.9, eps=1e-6)
    dev = (y.cuda(), res.cuda())
    more = dict(post_weight=post.cuda(), gate=gt.cuda(), pre_weight=pre.cuda(), route=_route_of(w, slot), **kw)
    got = _ops().block_norm_quant(*dev, **more)
    _check_block(got, M.block(y, res, post=post, gate=gt, pre=pre, weights=w, slot_row=slot, **kw), wide)
    again = _ops().block_norm_quant(*dev, **more)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, again))
    from fp8_hand_b200 import _native
    assert _native.status() == 0


@pytest.mark.parametrize("H", [640, 5120, 8192])
def test_block_scales_at_their_floor(cuda_lib, H):
    """Groups whose norm weight is so small that the scale is at its floor beside ordinary ones."""
    y, res, post, pre, _, _, _ = _block_case(7, H, 0, False, H)
    pre[:128] *= 1e-13
    pre[256:384] = 0
    pre[384:512] *= 1e-30
    got = _ops().block_norm_quant(y.cuda(), res.cuda(), post_weight=post.cuda(), pre_weight=pre.cuda())
    _check_block(got, M.block(y, res, post=post, pre=pre), False)
    floor = got[2] == torch.tensor(1e-12)
    assert bool(floor[:, [0, 2, 3]].all()) and not bool(floor[:, [1, 4]].any())


@pytest.mark.parametrize("k", [0, 4])
def test_block_plain_add_and_norm(cuda_lib, k):
    """No norm after the block and no gate: h = residual + z, then the next block's quant."""
    y, res, _, pre, w, slot, _ = _block_case(50, 1024, k, False, 4)
    got = _ops().block_norm_quant(y.cuda(), res.cuda(), pre_weight=pre.cuda(), route=_route_of(w, slot))
    _check_block(got, M.block(y, res, pre=pre, weights=w, slot_row=slot), False)


@pytest.mark.parametrize("k", [0, 3])
def test_block_without_residual_and_norm_out(cuda_lib, k):
    """h = scale * gate * n alone, and the bf16 norm beside its group quant."""
    y, res, post, pre, w, slot, g = _block_case(33, 768, k, False, 12)
    gt = torch.sigmoid(torch.randn(768, generator=g)).to(torch.bfloat16)
    h, A, As, v = _ops().block_norm_quant(y.cuda(), None, post_weight=post.cuda(), gate=gt.cuda(), scale=1.5,
                                          pre_weight=pre.cuda(), route=_route_of(w, slot), norm_out=True)
    want = M.block(y, torch.zeros_like(res), post=post, gate=gt, scale=1.5, pre=pre, weights=w, slot_row=slot)
    _check_block((h, A, As), want, False)
    _within(v, want[2], want[3], BF16_HALF)
    got = _ops().block_norm_quant(y.cuda(), None, route=_route_of(w, slot))
    _check_block(got, M.block(y, torch.zeros_like(res), weights=w, slot_row=slot), False)


def test_block_strides_and_zero_rows(cuda_lib):
    """Rows of wider tensors, odd starts (copied), a broadcast gate per token, all-zero rows, T = 0."""
    y, res, post, pre, _, _, g = _block_case(9, 384, 0, False, 6)
    y[4] = 0
    res[4] = 0
    bigy, bigr = torch.zeros(9, 600, dtype=torch.bfloat16), torch.zeros(9, 401, dtype=torch.bfloat16)
    bigy[:, 8:392], bigr[:, 3:387] = y, res
    gt = torch.rand(1, 1, generator=g).to(torch.bfloat16)
    out = torch.zeros(9, 512, dtype=torch.bfloat16, device="cuda")
    got = _ops().block_norm_quant(bigy.cuda()[:, 8:392], bigr.cuda()[:, 3:387], post_weight=post.cuda(),
                                  gate=gt.cuda().expand(9, 1), pre_weight=pre.cuda(), out=out[:, :384])
    _check_block(got, M.block(y, res, post=post, gate=gt.expand(9, 1), pre=pre), False)
    assert bool((out[:, 384:] == 0).all()) and bool((got[1][4].float() == 0).all()) and bool((got[2][4] == 1e-12).all())
    h, a, s = _ops().block_norm_quant(y.cuda()[:0], res.cuda()[:0], pre_weight=pre.cuda())
    assert h.shape == (0, 384) and a.shape == (0, 384) and s.shape == (0, 3)


def test_block_not_finite(cuda_lib):
    """A NaN or an infinity poisons its own token and no other."""
    y, res, post, pre, _, _, _ = _block_case(6, 512, 0, False, 8)
    y[1, 5], res[3, 9] = math.nan, math.inf
    got = _ops().block_norm_quant(y.cuda(), res.cuda(), post_weight=post.cuda(), pre_weight=pre.cuda())
    keep = [0, 2, 4, 5]
    want = M.block(y[keep], res[keep], post=post, pre=pre)
    _check_block(tuple(t[torch.tensor(keep, device="cuda")] if t.dtype != torch.float8_e4m3fn else
                       t.view(torch.uint8)[torch.tensor(keep, device="cuda")].view(torch.float8_e4m3fn) for t in got), want, False)
    assert bool(got[0][1].isnan().all()) and bool(got[1][1].float().isnan().all())
    assert math.isinf(float(got[0][3, 9])) and bool(got[1][3].float().isnan().any())


# ----------------------------------------------------------------------------- streams, graphs, refusals
def test_side_stream_and_graph(cuda_lib):
    """The chain on a stream of its own, and captured once and replayed on new inputs."""
    ops = _ops()
    T, E, k, H, inter = 20, 8, 2, 256, 128
    ws = [O.make_weight(2 * inter, H, e) for e in range(E)]
    B, Bs = torch.stack([w.view(torch.uint8) for w, _ in ws]).view(torch.float8_e4m3fn).cuda(), torch.stack([s for _, s in ws]).cuda()
    ws = [O.make_weight(H, inter, 50 + e) for e in range(E)]
    D, Ds = torch.stack([w.view(torch.uint8) for w, _ in ws]).view(torch.float8_e4m3fn).cuda(), torch.stack([s for _, s in ws]).cuda()
    pre = torch.ones(H, dtype=torch.bfloat16, device="cuda")

    def chain(x, logits):
        A, As = ops.group_quant(x)
        r = ops.moe_route(logits, k)
        Q, Qs = ops.grouped_gemm_silu_quant(A, B, As, Bs, r)
        y = ops.grouped_gemm(Q, D, Qs, Ds, r)
        return ops.block_norm_quant(y, x, pre_weight=pre, route=r)

    g = torch.Generator().manual_seed(1)
    ins = [(torch.randn(T, H, generator=g).to(torch.bfloat16).cuda(), torch.randn(T, E, generator=g).cuda()) for _ in range(2)]
    want = [chain(*i) for i in ins]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = chain(*ins[1])
    side.synchronize()
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want[1]))
    x, logits = ins[0][0].clone(), ins[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = chain(x, logits)
    for i, w in zip(ins, want):
        x.copy_(i[0])
        logits.copy_(i[1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(out, w))


def _experts(E, inter, H, seed):
    w13, s13 = zip(*[O.make_weight(2 * inter, H, seed + e) for e in range(E)])
    w2, s2 = zip(*[O.make_weight(H, inter, seed + 100 + e) for e in range(E)])
    stack = lambda ws: torch.stack([t.view(torch.uint8) for t in ws]).view(torch.float8_e4m3fn)  # noqa: E731
    return stack(w13), torch.stack(s13), stack(w2), torch.stack(s2)


@pytest.mark.parametrize("T", [1, 90])
def test_sparse_block(cuda_lib, monkeypatch, T):
    """The path that runs them together: two SparseBlocks, tile-first after post_load. Each stage is checked against the
    64-bit oracle on the stage's own inputs, expert halves on two ranks add up to the whole."""
    import fp8_hand_b200.fp8_hand_sm100 as hand
    from fp8_hand_b200 import sglang_compat as S
    monkeypatch.setattr(hand, "ENABLED", True)
    ops = _ops()
    E, k, H, inter = 6, 2, 512, 256
    w13, s13, w2, s2 = _experts(E, inter, H, 40)
    g = torch.Generator().manual_seed(T)
    bf = torch.bfloat16
    norms = [(1 + 0.1 * torch.randn(H, generator=g)).to(bf) for _ in range(4)]
    router = torch.randn(E, H, generator=g).to(bf)
    mlp = S.SparseMLP(w13.cuda(), s13.cuda(), w2.cuda(), s2.cuda(), k)
    block = S.SparseBlock(router.cuda(), mlp, norms[1].cuda(), post_norm=norms[2].cuda(), scale=0.5).cuda()
    x = torch.randn(T, H, generator=g).to(bf)
    state = S.SparseBlock.enter(x.cuda(), norms[0].cuda())
    row_major = block(*state)
    S.post_load(block)
    assert mlp.w13_weight.device.type == "meta" and mlp.w13_weight.tiles.shape == (E, 2 * inter // 128, H // 128, 128, 128)
    out = block(*state)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(out, row_major))
    # stage by stage
    h, A, As, v = state
    logits = torch.nn.functional.linear(v, router.cuda())
    rows, route = mlp.experts((A, As), logits)
    _check_route(route, logits.cpu(), k)
    off, src, _ = M.plan(route.ids.cpu(), 0, E)
    Q, Qs = ops.grouped_gemm_silu_quant(A, mlp.w13_weight.tiles, As, s13.cuda(), route, b_tiled=True)
    M.check_quant(Q.cpu(), Qs.cpu(), *M.silu_mul(*M.grouped(A.cpu(), As.cpu(), w13, s13, off, src)), 1e-10 / 448)
    _within(rows, *M.grouped(Q.cpu(), Qs.cpu(), w2, s2, off, torch.arange(T * k)), BF16_HALF)
    want = M.block(rows.cpu(), h.cpu(), post=norms[2], scale=0.5, pre=norms[1], weights=route.weights.cpu(),
                   slot_row=route.slot_row.cpu())
    _check_block(out[:3], want, False)
    block(*out)  # the stream goes on
    # two expert-parallel halves
    whole = mlp((A, As), logits)
    parts = [S.SparseMLP(w13[i:i + 3].cuda(), s13[i:i + 3].cuda(), w2[i:i + 3].cuda(), s2[i:i + 3].cuda(), k, first_expert=i)
             ((A, As), logits) for i in (0, 3)]
    # each half and the whole are rounded once to bf16
    lim = 2.0 ** -8 * 1.01 * (parts[0].abs() + parts[1].abs() + whole.abs()).double().cpu() + 1e-30
    assert bool(((parts[0].double() + parts[1].double() - whole.double()).abs().cpu() <= lim + 1e-6 * lim.max()).all())


def test_refusals(cuda_lib):
    ops = _ops()
    bf, dev = torch.bfloat16, "cuda"
    with pytest.raises(ValueError):
        ops.moe_route(torch.zeros(4, 8, dtype=torch.float16, device=dev), 2)
    with pytest.raises(ValueError):
        ops.moe_route(torch.zeros(4, 8, device=dev), 9)
    with pytest.raises(ValueError):
        ops.moe_route(torch.zeros(4, 513, device=dev), 2)
    with pytest.raises(ValueError):
        ops.moe_route(torch.zeros(4, 8, device=dev), 2, experts=(4, 5))
    with pytest.raises(ValueError):
        ops.moe_dispatch(torch.zeros(4, 2, dtype=torch.int64, device=dev), None, 8)
    r = ops.moe_route(torch.zeros(4, 2, device=dev), 1)
    A, As = ops.group_quant(torch.zeros(4, 256, dtype=bf, device=dev))
    B, Bs = torch.zeros(2, 256, 256, dtype=torch.uint8, device=dev), torch.ones(2, 2, 2, device=dev)
    for bad in (dict(B=B[:, :, :128]), dict(B=B[:1]), dict(Bs=Bs[:, :1]), dict(As=As[:, :1]), dict(A=A[:, :128]),
                dict(A=A.to(bf)), dict(B=B[:, :200].contiguous())):
        a = {**dict(A=A, B=B, As=As, Bs=Bs), **bad}
        with pytest.raises(ValueError):
            ops.grouped_gemm(a["A"], a["B"], a["As"], a["Bs"], r)
    with pytest.raises(ValueError):
        ops.grouped_gemm_silu_quant(A, B[:, :128].contiguous(), As, Bs[:, :1].contiguous(), r)
    with pytest.raises(ValueError):
        ops.grouped_gemm(A[:2], B, As[:2], Bs, r)
    with pytest.raises(ValueError):
        ops.grouped_gemm(A, B, As, Bs, r, out=torch.zeros(4, 128, device=dev))
    with pytest.raises(ValueError):
        ops.grouped_gemm(A.cpu(), B, As, Bs, r)
    y = torch.zeros(4, 256, dtype=bf, device=dev)
    for bad in (dict(residual=y[:3]), dict(residual=y.half()), dict(gate=y[:, :7]), dict(gate=y.float()),
                dict(post_weight=y[0, :128]), dict(pre_weight=y[0].float()), dict(out=y[:2]),
                dict(route=ops.moe_dispatch(r.ids, None, 2)), dict(y=y[:, :200])):
        a = {**dict(y=y, residual=y), **bad}
        with pytest.raises(ValueError):
            ops.block_norm_quant(a.pop("y"), a.pop("residual"), **a)
    assert bool((y == 0).all())


def test_refusals_of_too_few_rows(cuda_lib):
    """A route for more tokens than there are rows: the products of the tokens that are not there, and their sums."""
    ops = _ops()
    bf, dev = torch.bfloat16, "cuda"
    r = ops.moe_route(torch.zeros(5, 2, device=dev), 2)
    A, As = ops.group_quant(torch.zeros(5, 256, dtype=bf, device=dev))
    B, Bs = torch.zeros(2, 256, 256, dtype=torch.uint8, device=dev), torch.ones(2, 2, 2, device=dev)
    y, res = torch.zeros(10, 256, dtype=bf, device=dev), torch.zeros(5, 256, dtype=bf, device=dev)
    ops.grouped_gemm_silu_quant(A, B, As, Bs, r)
    ops.grouped_gemm(A, B, As, Bs, r, gather=True)
    ops.block_norm_quant(y, res, route=r)
    with pytest.raises(ValueError, match="A has 4 rows, the route has 5 tokens"):
        ops.grouped_gemm_silu_quant(A[:4], B, As[:4], Bs, r)
    with pytest.raises(ValueError, match="A has 4 rows, the route has 5 tokens"):
        ops.grouped_gemm(A[:4], B, As[:4], Bs, r, gather=True)
    with pytest.raises(ValueError, match="A has 5 rows, the route has 10 rows"):
        ops.grouped_gemm(A, B, As, Bs, r)
    with pytest.raises(ValueError, match="y has 9 rows, the route has 10"):
        ops.block_norm_quant(y[:9], res, route=r)
    with pytest.raises(ValueError, match="y has 0 rows"):
        ops.block_norm_quant(y[:0], None, route=r)


def test_output_stride_beyond_32_bits(cuda_lib):
    """Rows further apart than the C-ABI's 32-bit stride can say: refused, nothing written (the storage is 8.6 GB). A
    stride just below is right, with the second row past 2^31 bytes."""
    ops = _ops()
    ids, B, Bs, A, As = _case([2], 256, 256, 3)
    r = ops.moe_dispatch(ids.cuda(), None, 1)
    off, src, _ = M.plan(ids, 0, 1)
    dev = [t.cuda() for t in (A, B, As, Bs)]
    out = torch.empty_strided((2, 256), ((1 << 32) + 256, 1), dtype=torch.bfloat16, device="cuda")
    out.zero_()
    with pytest.raises(ValueError, match="row stride"):
        ops.grouped_gemm(*dev, r, gather=True, out=out)
    assert bool((out == 0).all())
    near = out.as_strided((2, 256), ((1 << 31) - 8, 1))
    ops.grouped_gemm(*dev, r, gather=True, out=near)
    _within(near, *M.grouped(A, As, B, Bs, off, src), BF16_HALF)
