"""A stack of mixture-of-experts blocks in block FP8, and its time per block.

    python examples/sparse_stack.py --tokens 64 --experts 64 --top-k 8 --hidden 2048 --inter 1024 --layers 4

Each block: router -> grouped gate_up + SiLU*up + quant -> grouped down -> weighted sum, norm, residual, next block's norm
and quant (fp8_hand_b200.sglang_compat.SparseBlock), with random weights. The stack is captured into one CUDA graph, as a
decode loop would, and replayed; --eager times the calls themselves.
"""
from __future__ import annotations

import argparse
import os
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "ucloud-ai-infra_b200"))
os.environ.setdefault("SGLANG_FP8_HAND_GEMM", "1")  # post_load moves the weights to tile-first storage

import torch  # noqa: E402

from fp8_hand_b200 import sglang_compat as S  # noqa: E402


def expert_weights(E: int, N: int, K: int, gen: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """N(0, 0.02) weights e4m3 [E, N, K] with a scale for each 128 x 128 block."""
    q = torch.empty((E, N, K), dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty((E, N // 128, K // 128), device="cuda")
    for e in range(E):
        w = torch.randn((N // 128, 128, K // 128, 128), generator=gen, device="cuda") * 0.02
        s[e] = (w.abs().amax((1, 3)) / 448).clamp_min(1e-12)
        q[e] = (w / s[e][:, None, :, None]).reshape(N, K).to(torch.float8_e4m3fn)
    return q, s


def build(a: argparse.Namespace, gen: torch.Generator) -> torch.nn.ModuleList:
    bf = torch.bfloat16
    blocks = torch.nn.ModuleList()
    for _ in range(a.layers):
        mlp = S.SparseMLP(*expert_weights(a.experts, 2 * a.inter, a.hidden, gen),
                          *expert_weights(a.experts, a.hidden, a.inter, gen), top_k=a.top_k)
        router = (torch.randn((a.experts, a.hidden), generator=gen, device="cuda") * 0.02).to(bf)
        ones = torch.ones(a.hidden, dtype=bf, device="cuda")
        blocks.append(S.SparseBlock(router, mlp, next_norm=ones, post_norm=ones))
    S.post_load(blocks)
    return blocks


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("tokens", 64), ("experts", 64), ("top-k", 8), ("hidden", 2048), ("inter", 1024), ("layers", 4),
                          ("iters", 20)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--eager", action="store_true", help="time the calls, not a captured graph")
    a = ap.parse_args(argv)
    gen = torch.Generator(device="cuda").manual_seed(0)
    with torch.inference_mode():
        blocks = build(a, gen)
        x = torch.randn((a.tokens, a.hidden), generator=gen, device="cuda").to(torch.bfloat16)
        first = torch.ones(a.hidden, dtype=torch.bfloat16, device="cuda")

        def run():
            state = S.SparseBlock.enter(x, first)
            for block in blocks:
                state = block(*state)
            return state[0]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            run()
        side.synchronize()
        step, graph = run, None
        if not a.eager:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = run()
            step = graph.replay
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        step()
        torch.cuda.synchronize()
        begin.record()
        for _ in range(a.iters):
            step()
        end.record()
        torch.cuda.synchronize()
        if a.eager:
            out = run()
        us = begin.elapsed_time(end) * 1e3 / a.iters / a.layers
        print(f"{a.tokens} tokens, {a.experts} experts, top {a.top_k}, {a.hidden} -> {a.inter}: {us:.1f} us per block "
              f"({'eager' if a.eager else 'graph'}), output rms {out.float().square().mean().sqrt():.3f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
