"""Stand-ins for the SGLang call sites the reference hooks into (SGLang 0.5.22 is not part of this
repository). They reproduce the three hook points of patches/apply_sglang_fp8_hand_gemm.py so the
drop-in module is exercised exactly as SGLang would call it:

  w8a8_block_fp8_matmul(A, B, As, Bs, block_size, output_dtype)   GEMM entry; the reference's hook
      `if fp8_hand_sm89.matmul(A, B, C, As, Bs, M, N, K, block_size): return C` sits after C is
      allocated (:26-33). Weights that were not relayouted run this library's row-major kernel
      where SGLang would run Triton.
  Fp8BlockLinear.forward(x)                                       Fp8LinearMethod.apply: activation
      quant then the GEMM entry; a pre-quantised (q, scale) tuple skips the quant, which is how
      the fused output reaches down_proj (:50-53).
  GatedMLP.forward(x)                                             the patched MLP forward (:45-56).
  post_load(model)                                                the loader hook (:59-65).

The same block as a mixture of experts, for which the reference has no counterpart (its models are dense):

  SparseMLP            the expert weights under the parameter names of SGLang's FusedMoE; routed products and their sum
  SparseBlock          norm -> router -> experts -> norm, gate and residual, handing the next block its quantised input
"""
from __future__ import annotations

import torch
from torch import nn

from . import fp8_hand_sm100 as fp8_hand
from . import ops

BLOCK = 128


def per_token_group_quant_fp8(x: torch.Tensor, group_size: int = BLOCK):
    """SGLang's activation quant entry (called at H:690-693): (A e4m3, As fp32 [..., K/128])."""
    return ops.group_quant(x, group_size)


def w8a8_block_fp8_matmul(A, B, As, Bs, block_size, output_dtype=torch.bfloat16):
    """SGLang's block-FP8 GEMM entry with the reference's hook in place."""
    N, K = B.shape
    M = A.numel() // A.shape[-1]
    C = torch.empty((*A.shape[:-1], N), dtype=output_dtype, device=A.device)
    if fp8_hand.matmul(A, B, C, As, Bs, M, N, K, block_size):
        return C
    if list(block_size) != [BLOCK, BLOCK]:
        raise ValueError(f"block_size {block_size}: only [128, 128] weight blocks exist on this path")
    return ops.gemm(A, B, As, Bs, b_tiled=False, out=C, out_dtype=output_dtype)


class Fp8BlockLinear(nn.Module):
    """Linear layer with block-FP8 weights, the shape of SGLang's Fp8LinearMethod-backed linear:
    weight e4m3 [N, K], weight_scale_inv fp32 [N/128, K/128]; forward returns (out, bias)."""

    def __init__(self, weight: torch.Tensor, weight_scale_inv: torch.Tensor, bias: torch.Tensor | None = None):
        super().__init__()
        self.weight = nn.Parameter(weight, requires_grad=False)
        self.weight_scale_inv = nn.Parameter(weight_scale_inv, requires_grad=False)
        self.bias = bias

    def forward(self, x):
        if isinstance(x, tuple):
            q, s = x
            out_dtype = torch.bfloat16
        else:
            q, s = per_token_group_quant_fp8(x.view(-1, x.shape[-1]), BLOCK)
            out_dtype = x.dtype
        out = w8a8_block_fp8_matmul(q, self.weight, s, self.weight_scale_inv, [BLOCK, BLOCK], out_dtype)
        if not isinstance(x, tuple):
            out = out.view(*x.shape[:-1], -1)
        return out, self.bias


def silu_and_mul(gate_up: torch.Tensor) -> torch.Tensor:
    """The unfused chain's activation (SGLang silu_and_mul): only reached when the fused kernel is
    switched off (SGLANG_FP8_HAND_FUSED=0) or ineligible. Runs the library's kernel (bs_fp8_silu_mul)."""
    from . import ops
    return ops.silu_mul(gate_up)


class GatedMLP(nn.Module):
    """gate_up_proj -> SiLU(gate) * up -> down_proj with the reference's patched forward."""

    def __init__(self, gate_up_proj: Fp8BlockLinear, down_proj: Fp8BlockLinear):
        super().__init__()
        self.gate_up_proj = gate_up_proj
        self.down_proj = down_proj

    def forward(self, x):
        fused = fp8_hand.fused_gate_up(self.gate_up_proj, x)
        if fused is not None:
            x, _ = self.down_proj(fused)
            return x
        gate_up, _ = self.gate_up_proj(x)
        x, _ = self.down_proj(silu_and_mul(gate_up))
        return x


class SparseMLP(nn.Module):
    """Gated MLP as a mixture of block-FP8 experts, under the parameter names of SGLang's FusedMoE:
    w13_weight e4m3 [E, 2I, H] (gate rows, then up rows) with w13_weight_scale_inv fp32 [E, 2I/128, H/128], and
    w2_weight e4m3 [E, H, I] with w2_weight_scale_inv. After post_load the weights are tile-first (their parameters stay
    on the meta device and carry `.tiles`). E are the experts held here, numbers first_expert .. first_expert + E - 1
    of the router's (expert parallelism: the ranks' outputs add up)."""

    expert_tiles = True  # relayout may move w13_weight and w2_weight

    def __init__(self, w13_weight: torch.Tensor, w13_weight_scale_inv: torch.Tensor, w2_weight: torch.Tensor,
                 w2_weight_scale_inv: torch.Tensor, top_k: int, *, renormalize: bool = True, routed_scale: float = 1.0,
                 first_expert: int = 0):
        super().__init__()
        self.w13_weight = nn.Parameter(w13_weight, requires_grad=False)
        self.w13_weight_scale_inv = nn.Parameter(w13_weight_scale_inv, requires_grad=False)
        self.w2_weight = nn.Parameter(w2_weight, requires_grad=False)
        self.w2_weight_scale_inv = nn.Parameter(w2_weight_scale_inv, requires_grad=False)
        self.top_k, self.renormalize, self.routed_scale = top_k, renormalize, routed_scale
        self.first_expert = first_expert

    def experts(self, x, router_logits: torch.Tensor) -> tuple[torch.Tensor, ops.MoeRoute]:
        """x bf16 [T, H] or its group quant (A, As) -> (the experts' rows bf16 [T * top_k, H], the route)."""
        A, As = x if isinstance(x, tuple) else ops.group_quant(x, BLOCK)
        route = ops.moe_route(router_logits, self.top_k, renormalize=self.renormalize, scale=self.routed_scale,
                              experts=(self.first_expert, self.w13_weight.shape[0]))
        w13, w2 = (getattr(w, "tiles", None) for w in (self.w13_weight, self.w2_weight))
        q, s = ops.grouped_gemm_silu_quant(A, self.w13_weight if w13 is None else w13, As, self.w13_weight_scale_inv, route,
                                           b_tiled=w13 is not None)
        rows = ops.grouped_gemm(q, self.w2_weight if w2 is None else w2, s, self.w2_weight_scale_inv, route,
                                b_tiled=w2 is not None)
        return rows, route

    def forward(self, x, router_logits: torch.Tensor) -> torch.Tensor:
        """sum over a token's slots of weight * expert(x): bf16 [T, H]."""
        rows, route = self.experts(x, router_logits)
        return ops.block_norm_quant(rows, None, route=route)


class SparseBlock(nn.Module):
    """A mixture-of-experts block between its norms. The stream between blocks is (h, A, As, v): the residual, the group
    quant of its norm (the experts' input) and the norm in bf16 (the router's). One call takes this block's
    (h, A, As, v) to the next's, whose norm weight is next_norm:
      h' = residual_scale * h + scale * gate * rmsnorm(experts(A, As; router(v))) * post_norm
    mlp holds every expert of the router: the norms need the sum over all of them, so a rank that holds some takes
    SparseMLP.forward, adds the ranks' outputs, and ends the block with ops.block_norm_quant on the sum."""

    def __init__(self, router_weight: torch.Tensor, mlp: SparseMLP, next_norm: torch.Tensor,
                 post_norm: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
                 residual_scale: float = 1.0, eps: float = 1e-6):
        super().__init__()
        if mlp.first_expert != 0 or mlp.w13_weight.shape[0] != router_weight.shape[0]:
            raise ValueError("a block's mlp must hold every expert of its router")
        self.router_weight = nn.Parameter(router_weight, requires_grad=False)
        self.mlp = mlp
        self.next_norm = nn.Parameter(next_norm, requires_grad=False)
        self.post_norm = None if post_norm is None else nn.Parameter(post_norm, requires_grad=False)
        self.gate = None if gate is None else nn.Parameter(gate, requires_grad=False)
        self.scale, self.residual_scale, self.eps = scale, residual_scale, eps

    @staticmethod
    def enter(x: torch.Tensor, norm: torch.Tensor, eps: float = 1e-6):
        """(h, A, As, v) of a stack's first block from the embeddings x bf16 [T, H]."""
        _, A, As, v = ops.block_norm_quant(x, None, pre_weight=norm, eps=eps, norm_out=True)
        return x, A, As, v

    def forward(self, h, A, As, v):
        logits = nn.functional.linear(v, self.router_weight)
        rows, route = self.mlp.experts((A, As), logits)
        return ops.block_norm_quant(rows, h, post_weight=self.post_norm, gate=self.gate, scale=self.scale,
                                    residual_scale=self.residual_scale, pre_weight=self.next_norm, eps=self.eps,
                                    route=route, norm_out=True)


def post_load(model: nn.Module, cache=None) -> None:
    """Loader post-hook (apply_sglang_fp8_hand_gemm.py:59-65): tile-first pre-pack, read from the
    tile-pack file `cache` when it exists (written there otherwise)."""
    fp8_hand.relayout(model, cache=cache)
