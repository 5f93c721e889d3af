"""CPU: argument checks of the mixture-of-experts entry points (refused before any GPU work) and the oracle's plan."""
import pytest
import torch

from oracle import moe as M


@pytest.fixture(scope="module")
def lib():
    from fp8_hand_b200 import _build, _native
    _build.build()
    return _native.lib()


P = 1 << 20  # a 16-byte aligned address that is never used: every call below is refused first


def test_route_arguments(lib):
    ok = dict(logits=P, dtype=0, ldl=64, T=4, E=64, k=8, renorm=1, scale=1.0, begin=0, count=64, w=P, ids=P, off=P, rt=P,
              sr=P, scratch=None, nbytes=0)

    def call(**kw):
        return lib.bs_fp8_moe_route(*{**ok, **kw}.values(), None)

    for bad in (dict(dtype=2), dict(ldl=63), dict(T=-1), dict(E=513, ldl=600), dict(k=0), dict(k=33), dict(k=9, E=8, count=8),
                dict(begin=-1), dict(begin=1), dict(count=0), dict(w=None), dict(ids=None), dict(off=None), dict(rt=None),
                dict(sr=None), dict(logits=None), dict(T=1 << 30)):
        assert call(**bad) == 1, bad
    assert call(dtype=1, logits=P + 2) == 2


def test_dispatch_arguments(lib):
    ok = dict(ids=P, T=4, E=64, k=8, begin=0, count=64, off=P, rt=P, sr=P, scratch=None, nbytes=0)
    for bad in (dict(ids=None), dict(E=0), dict(k=33), dict(begin=60, count=5), dict(off=None), dict(sr=None)):
        assert lib.bs_fp8_moe_dispatch(*{**ok, **bad}.values(), None) == 1, bad


def test_scratch_bytes(lib):
    assert lib.bs_fp8_moe_scratch_bytes(0, 64) == 0 and lib.bs_fp8_moe_scratch_bytes(1, 64) == 0
    big = lib.bs_fp8_moe_scratch_bytes(8192, 64)
    assert big > 0 and big % (64 * 4) == 0


def test_grouped_arguments(lib):
    ok = dict(A=P, B=P, C=P, As=P, Bs=P, off=P, rt=None, rows_a=64, R=64, hint=0, E=8, N=256, K=256, ldc=256, tiled=0, dt=0)

    def call(**kw):
        return lib.bs_fp8_grouped_gemm(*{**ok, **kw}.values(), None)

    for bad in (dict(K=200), dict(N=200), dict(ldc=128), dict(ldc=260), dict(dt=2), dict(tiled=2), dict(E=0), dict(E=513),
                dict(rows_a=63), dict(rows_a=0, rt=P), dict(hint=65), dict(R=-1), dict(off=None), dict(A=None), dict(Bs=None),
                dict(E=512, N=1 << 22, K=128, ldc=1 << 22)):
        assert call(**bad) == 1, bad
    assert call(B=P + 8) == 2 and call(C=P + 4) == 2
    assert call(R=0, rows_a=0, A=None, B=None, C=None, As=None, Bs=None, off=None) == 0
    fused = dict(A=P, B=P, Q=P, As=P, Bs=P, Qs=P, off=P, rt=P, rows_a=8, R=64, hint=0, E=8, N2=512, K=256, tiled=1)
    for bad in (dict(N2=384), dict(Qs=None), dict(K=0), dict(tiled=-1)):
        assert lib.bs_fp8_grouped_gemm_silu_quant(*{**fused, **bad}.values(), None) == 1, bad


# rows expected, experts, N (N2), K, fused -> kind, rows per tile, CTAs per tile, on 148 SMs (or as many as are there)
GROUPED_PLANS = [
    ((8, 64, 2048, 5120, True), (1, 16, 2)),      # one token: 64 tiles
    ((488, 64, 2048, 5120, True), (1, 32, 2)),    # more tiles than SMs, fused: two CTAs per tile
    ((488, 64, 5120, 1024, False), (1, 32, 1)),   # plain: one
    ((1025, 64, 2048, 5120, True), (2, 128, 1)),  # more than 16 rows per expert
    ((897, 64, 5120, 1024, False), (2, 128, 1)),  # more than 14
    ((4, 1, 256, 1920, False), (1, 16, 1)),       # fewer than 16 K blocks
    ((4, 1, 256, 2048, False), (1, 16, 2)),
    ((5, 1, 256, 4096, False), (1, 32, 4)),
    ((5, 1, 512, 8192, True), (1, 32, 8)),
    ((5, 1, 512, 65536, True), (1, 32, 8)),
]


@pytest.mark.parametrize("shape,want", GROUPED_PLANS)
def test_grouped_plan(lib, shape, want):
    from fp8_hand_b200 import _native
    if _native.num_sms() not in (0, 148):
        pytest.skip("the rule goes by the number of SMs")
    assert tuple(_native.grouped_plan(*shape).values()) == want


def test_grouped_plan_arguments(lib):
    from fp8_hand_b200 import _native
    for bad in ((0, 1, 256, 256, False), (4, 0, 256, 256, False), (4, 513, 256, 256, False), (4, 1, 200, 256, False),
                (4, 1, 384, 256, True), (4, 1, 256, 200, False)):
        with pytest.raises(RuntimeError):
            _native.grouped_plan(*bad)
    assert lib.bs_fp8_grouped_plan(4, 1, 256, 256, 0, None, 3) == 1


def test_block_arguments(lib):
    ok = dict(y=P, ldy=256, rows=4, w=None, sr=None, k=0, res=P, ldr=256, out=P, ldo=256, wide=0, post=None, gate=None, kind=0,
              ldg=0, scale=1.0, rscale=1.0, pre=P, eps=1e-6, A=P, As=P, V=None, T=4, H=256)

    def call(**kw):
        return lib.bs_fp8_block_norm_quant(*{**ok, **kw}.values(), None)

    for bad in (dict(H=200), dict(H=16512, ldy=16512, ldr=16512, ldo=16512), dict(ldy=128), dict(ldy=260), dict(ldr=258),
                dict(ldo=250), dict(wide=2), dict(eps=-1.0), dict(eps=float("nan")), dict(kind=1), dict(gate=P), dict(kind=4, gate=P),
                dict(kind=3, gate=P, ldg=128), dict(kind=2, gate=P, ldg=0), dict(w=P), dict(w=P, sr=P), dict(rows=3), dict(T=-1),
                dict(A=None), dict(V=P, pre=None), dict(w=P, sr=P, k=33)):
        assert call(**bad) == 1, bad
    assert call(y=P + 2) == 2 and call(pre=P + 8) == 2 and call(kind=1, gate=P + 2) == 2
    assert call(T=0, rows=0) == 0


def test_oracle_plan_is_a_stable_sort():
    ids = torch.tensor([[2, 0], [0, -1], [2, 2], [5, 1]], dtype=torch.int32)
    off, row_token, slot_row = M.plan(ids, 0, 3)
    assert off.tolist() == [0, 2, 3, 6]
    assert row_token.tolist() == [0, 1, 3, 0, 2, 2, -1, -1]
    assert slot_row.tolist() == [[3, 0], [1, -1], [4, 5], [-1, 2]]


def test_host_tensors_are_refused():
    from fp8_hand_b200 import ops
    with pytest.raises(ValueError):
        ops.moe_route(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError):
        ops.block_norm_quant(torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(4, 128, dtype=torch.bfloat16))


# ----------------------------------------------------------------------------- weights at load
def _expert_parameters(module, E=2, inter=128, H=256, device="cpu"):
    for name, n, k in (("w13_weight", 2 * inter, H), ("w2_weight", H, inter)):
        w = torch.arange(E * n * k, dtype=torch.int32).remainder(97).to(torch.uint8).view(torch.float8_e4m3fn).view(E, n, k)
        setattr(module, name, torch.nn.Parameter(w.to(device), requires_grad=False))
        scale = torch.ones(E, n // 128, k // 128)
        setattr(module, name + "_scale_inv", torch.nn.Parameter(scale, requires_grad=False))
    return module


@pytest.fixture
def hand(monkeypatch):
    """The drop-in module as it runs on a B200, with the oracle's permute in place of the packing kernel."""
    import fp8_hand_b200.fp8_hand_sm100 as hand
    from oracle import oracle as O
    monkeypatch.setattr(hand, "ENABLED", True)
    monkeypatch.setattr(hand, "_is_b200", lambda: True)
    monkeypatch.setattr(hand.ops, "pack_tiles", lambda w: O.relayout_tiles(w.view(torch.uint8)))
    return hand


def test_relayout_leaves_foreign_experts(hand):
    """A module that has the parameter names but reads the row-major weights itself (SGLang's FusedMoE) keeps them."""
    class FusedMoE(torch.nn.Module):
        pass

    moe = _expert_parameters(FusedMoE())
    on_meta = _expert_parameters(FusedMoE(), device="meta")
    kept = {k: v.clone() for k, v in moe.named_parameters()}
    hand.relayout(torch.nn.ModuleList([moe, on_meta]))
    for k, v in moe.named_parameters():
        assert v.device.type == "cpu" and torch.equal(v.view(torch.uint8), kept[k].view(torch.uint8)), k
    assert not any(hasattr(p, "tiles") for m in (moe, on_meta) for p in m.parameters())


def test_relayout_moves_sparse_mlp(hand):
    from fp8_hand_b200 import sglang_compat as S
    src = _expert_parameters(torch.nn.Module())
    mlp = S.SparseMLP(src.w13_weight.data, src.w13_weight_scale_inv.data, src.w2_weight.data, src.w2_weight_scale_inv.data, 1)
    hand.relayout(torch.nn.Sequential(mlp))
    assert mlp.w13_weight.device.type == mlp.w2_weight.device.type == "meta"
    bytes13 = src.w13_weight.data.view(torch.uint8)
    assert mlp.w13_weight.tiles.shape == (2, 2, 2, 128, 128)
    assert torch.equal(mlp.w13_weight.tiles[1, 1, 0].view(torch.uint8), bytes13[1, 128:, :128])
    assert hand.relayout_experts(mlp) == 0  # a second call finds nothing to do
    del mlp.w13_weight.tiles
    with pytest.raises(hand.tilepack.TilePackError, match="w13_weight: weight not loaded"):
        hand.relayout(mlp)


@pytest.mark.parametrize("experts,first,ok", [(4, 0, True), (2, 0, False), (2, 2, False), (4, 4, False), (6, 0, False)])
def test_sparse_block_needs_every_expert(experts, first, ok):
    """The norms are not linear: a block over some of the experts would normalise a partial sum."""
    from fp8_hand_b200 import sglang_compat as S
    src = _expert_parameters(torch.nn.Module(), E=experts)
    mlp = S.SparseMLP(src.w13_weight.data, src.w13_weight_scale_inv.data, src.w2_weight.data, src.w2_weight_scale_inv.data, 1,
                      first_expert=first)
    norm, router = torch.ones(256, dtype=torch.bfloat16), torch.zeros(4, 256, dtype=torch.bfloat16)
    if ok:
        S.SparseBlock(router, mlp, norm)
    else:
        with pytest.raises(ValueError, match="every expert"):
            S.SparseBlock(router, mlp, norm)


@pytest.mark.parametrize("T,k", [((1 << 30) + 1, 1), (1 << 28, 5), (1 << 32, 1), ((1 << 32) + 4, 8)])
def test_row_counts_beyond_32_bits_are_refused(T, k):
    """Sizes that would wrap in the C-ABI's 32-bit arguments (2^32 tokens would be none)."""
    from fp8_hand_b200 import ops
    with pytest.raises(ValueError, match="rows"):
        ops.moe_route(torch.zeros(1, 16).expand(T, 16), k)
    with pytest.raises(ValueError, match="rows"):
        ops.moe_dispatch(torch.zeros(1, k, dtype=torch.int32).expand(T, k), None, 16)
