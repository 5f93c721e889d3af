"""Tensor-level entry points over the C-ABI: activation quant, weight pre-pack, block-scaled FP8
GEMM and the fused gate_up + SiLU*up + quant front half.

All functions take CUDA tensors, launch on the current stream of the tensors' device, never
synchronise and never fall back: a tensor outside the contract raises ValueError, a library
failure raises RuntimeError.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native

E4M3 = torch.float8_e4m3fn
BLOCK = 128
MAX_EXPERTS = 512
MAX_TOP_K = 32


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _cuda(*ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    for t in ts:
        _need(t.is_cuda, "tensors must be on a CUDA device (this path has no CPU implementation)")
        _need(t.device == dev, "all tensors must be on the same device")
    return dev


def _as_bytes(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.uint8 else t.view(torch.uint8)


def group_quant(x: torch.Tensor, group_size: int = BLOCK) -> tuple[torch.Tensor, torch.Tensor]:
    """x bf16 [..., K] -> (A e4m3 [..., K], As fp32 [..., K/128]); per 1x128 group
    As = max(amax/448, 1e-12), A = e4m3(x / As)."""
    _need(group_size == BLOCK, "only 128-wide groups are supported")
    _need(x.dtype == torch.bfloat16, "x must be bf16")
    dev = _cuda(x)
    K = x.shape[-1]
    _need(K % BLOCK == 0, "K must be a multiple of 128")
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    M = x2.shape[0]
    A = torch.empty((M, K), dtype=E4M3, device=dev)
    As = torch.empty((M, K // BLOCK), dtype=torch.float32, device=dev)
    with _native.device_guard(dev):
        _native.check(_native.lib().bs_fp8_group_quant(
            x2.data_ptr(), x2.stride(0), A.data_ptr(), As.data_ptr(), M, K, _native.stream_handle(dev)),
            "bs_fp8_group_quant")
    return A.view(*x.shape[:-1], K), As.view(*x.shape[:-1], K // BLOCK)


def silu_mul(gate_up: torch.Tensor) -> torch.Tensor:
    """gate_up bf16 [..., 2I] -> bf16 [..., I]: silu(g) * u in fp32 with one rounding (SGLang's silu_and_mul,
    the unfused chain's activation)."""
    _need(gate_up.dtype == torch.bfloat16, "gate_up must be bf16")
    dev = _cuda(gate_up)
    n2 = gate_up.shape[-1]
    _need(n2 % 16 == 0, "gate_up width must be a multiple of 16")
    x2 = gate_up.reshape(-1, n2)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    M, inter = x2.shape[0], n2 // 2
    y = torch.empty((M, inter), dtype=torch.bfloat16, device=dev)
    with _native.device_guard(dev):
        _native.check(_native.lib().bs_fp8_silu_mul(
            x2.data_ptr(), x2.stride(0), y.data_ptr(), inter, M, inter, _native.stream_handle(dev)),
            "bs_fp8_silu_mul")
    return y.view(*gate_up.shape[:-1], inter)


def rmsnorm_group_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                        residual: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm fused with the per-token-group quant of its output (the next linear's activation quant):
    h = x, or h = bf16(x + residual) stored into `residual` in place (fused add); y = bf16(h * rsqrt(mean(h^2)
    + eps) * weight); returns group_quant(y) = (A e4m3 [..., K], As fp32 [..., K/128]) without storing y."""
    _need(x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16, "x and weight must be bf16")
    dev = _cuda(x, weight) if residual is None else _cuda(x, weight, residual)
    K = x.shape[-1]
    _need(K % BLOCK == 0, "K must be a multiple of 128")
    _need(weight.shape == (K,) and weight.is_contiguous(), "weight must be contiguous [K]")
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    M = x2.shape[0]
    r_ptr, ldr = None, K
    if residual is not None:
        _need(residual.dtype == torch.bfloat16 and residual.shape == x.shape, "residual must be bf16 like x")
        r2 = residual.view(-1, K)
        _need(r2.stride(-1) == 1 and r2.stride(0) % 8 == 0 and r2.data_ptr() % 16 == 0,
              "residual rows must be contiguous and 16-byte aligned (it is updated in place)")
        r_ptr, ldr = r2.data_ptr(), r2.stride(0)
    A = torch.empty((M, K), dtype=E4M3, device=dev)
    As = torch.empty((M, K // BLOCK), dtype=torch.float32, device=dev)
    with _native.device_guard(dev):
        _native.check(_native.lib().bs_fp8_rmsnorm_group_quant(
            x2.data_ptr(), x2.stride(0), r_ptr, ldr, weight.data_ptr(), float(eps), A.data_ptr(), As.data_ptr(),
            M, K, _native.stream_handle(dev)), "bs_fp8_rmsnorm_group_quant")
    return A.view(*x.shape[:-1], K), As.view(*x.shape[:-1], K // BLOCK)


def pack_tiles(weight: torch.Tensor) -> torch.Tensor:
    """e4m3 weight [N, K] -> tile-first bytes [N/128, K/128, 128, 128] (H:667 layout)."""
    _need(weight.dim() == 2 and weight.dtype in (E4M3, torch.uint8), "weight must be e4m3 [N, K]")
    dev = _cuda(weight)
    N, K = weight.shape
    _need(N % BLOCK == 0 and K % BLOCK == 0, "N and K must be multiples of 128")
    w = _as_bytes(weight.contiguous())
    tiles = torch.empty((N // BLOCK, K // BLOCK, BLOCK, BLOCK), dtype=torch.uint8, device=dev)
    with _native.device_guard(dev):
        _native.check(_native.lib().bs_fp8_pack_tiles(w.data_ptr(), tiles.data_ptr(), N, K,
                                                      _native.stream_handle(dev)), "bs_fp8_pack_tiles")
    return tiles


def _weight_geometry(B: torch.Tensor, b_tiled: bool) -> tuple[int, int]:
    if b_tiled:
        _need(B.dim() == 4 and tuple(B.shape[2:]) == (BLOCK, BLOCK) and B.dtype in (torch.uint8, E4M3),
              "tile-first weights must be [N/128, K/128, 128, 128] bytes")
        return B.shape[0] * BLOCK, B.shape[1] * BLOCK
    _need(B.dim() == 2 and B.dtype in (E4M3, torch.uint8), "row-major weights must be e4m3 [N, K]")
    return B.shape[0], B.shape[1]


def _check_operands(A, B, As, Bs, b_tiled):
    _need(A.dtype in (E4M3, torch.uint8), "A must be e4m3")
    dev = _cuda(A, B, As, Bs)
    N, K = _weight_geometry(B, b_tiled)
    _need(A.shape[-1] == K, f"A has K={A.shape[-1]}, weights have K={K}")
    A2 = A.reshape(-1, K)
    M = A2.shape[0]
    _need(As.dtype == torch.float32 and Bs.dtype == torch.float32, "scales must be fp32")
    _need(As.numel() == M * (K // BLOCK), "As must be [M, K/128]")
    _need(tuple(Bs.shape) == (N // BLOCK, K // BLOCK), "Bs must be [N/128, K/128]")
    _need(B.is_contiguous(), "weights must be contiguous")
    if not A2.is_contiguous():
        A2 = A2.contiguous()
    return dev, A2, As.reshape(M, K // BLOCK).contiguous(), Bs.contiguous(), M, N, K


def gemm(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, *, b_tiled: bool = False,
         out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C[m, n] = sum_kb (A . B)[m, n, kb] * As[m, kb] * Bs[n/128, kb] -> out [..., N] (bf16 or fp32)."""
    dev, A2, As2, Bs2, M, N, K = _check_operands(A, B, As, Bs, b_tiled)
    if out is None:
        out = torch.empty((*A.shape[:-1], N), dtype=out_dtype, device=dev)
    _need(out.dtype in (torch.bfloat16, torch.float32), "output must be bf16 or fp32")
    _need(out.device == dev and out.shape[-1] == N and out.numel() == M * N, "output must be [..., N]")
    out2 = out.view(M, N)
    _need(out2.stride(-1) == 1, "output rows must be contiguous")
    ldc = out2.stride(0) if M > 1 else N
    lib = _native.lib()
    with _native.device_guard(dev):
        ws_bytes = lib.bs_fp8_workspace_bytes(M, N, K, 0)
        ws = _native.workspace(dev, ws_bytes)
        _native.check(lib.bs_fp8_gemm(
            A2.data_ptr(), _as_bytes(B).data_ptr(), out2.data_ptr(), As2.data_ptr(), Bs2.data_ptr(), M, N, K, ldc,
            int(b_tiled), 0 if out.dtype == torch.bfloat16 else 1, _native.ptr(ws),
            0 if ws is None else ws.numel(), _native.stream_handle(dev)), "bs_fp8_gemm")
    return out


def gemm_reduce_multicast(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, out: torch.Tensor,
                          out_multicast: int, *, b_tiled: bool = False) -> torch.Tensor:
    """Row-parallel GEMM fused with the tensor-parallel sum: this rank's bf16 product is added into every
    rank's copy of `out` through the NVSwitch multicast address `out_multicast` (the address of out[0, 0] in
    the group's multicast mapping). `out` is this rank's copy, bf16 [M, N]; every rank zeroes its copy and
    the group synchronises before the call, and again before `out` is read."""
    dev, A2, As2, Bs2, M, N, K = _check_operands(A, B, As, Bs, b_tiled)
    _need(out.dtype == torch.bfloat16, "output must be bf16 (the switch adds bf16 pairs)")
    _need(out.device == dev and out.dim() == 2 and tuple(out.shape) == (M, N), "output must be [M, N]")
    _need(out.stride(-1) == 1, "output rows must be contiguous")
    _need(isinstance(out_multicast, int) and out_multicast != 0, "a multicast address is required")
    ldc = out.stride(0) if M > 1 else N
    lib = _native.lib()
    with _native.device_guard(dev):
        ws_bytes = lib.bs_fp8_workspace_bytes(M, N, K, 0)
        ws = _native.workspace(dev, ws_bytes)
        _native.check(lib.bs_fp8_gemm_reduce_multicast(
            A2.data_ptr(), _as_bytes(B).data_ptr(), out_multicast, As2.data_ptr(), Bs2.data_ptr(), M, N, K, ldc,
            int(b_tiled), _native.ptr(ws), 0 if ws is None else ws.numel(), _native.stream_handle(dev)),
            "bs_fp8_gemm_reduce_multicast")
    return out


def tp_reduce_switch(data: torch.Tensor, data_multicast: int, flags: torch.Tensor, flags_multicast: int, rank: int,
                     world: int, epoch: int, limit_ns: int = 0) -> torch.Tensor:
    """In-place tensor-parallel sum of the ranks' bf16 partials through the NVSwitch. `data` is this rank's copy
    of a symmetric bf16 buffer (contiguous, holding its partial) and `data_multicast` the multicast address of
    data's first element; `flags` this rank's copy of a symmetric int32 buffer of flag_words(world) words zeroed
    before the first call, `flags_multicast` its multicast address. Every rank calls with the same epoch (1, 2,
    ... per call on these flags). On return every rank's `data` holds the same sums."""
    dev = _cuda(data, flags)
    _need(data.dtype == torch.bfloat16 and data.is_contiguous(), "data must be contiguous bf16")
    _need(flags.dtype == torch.int32 and flags.numel() >= tp_flag_words(world), "flags too small for this world")
    _need(data.numel() % 8 == 0, "data must hold a multiple of 8 elements")
    lib = _native.lib()
    with _native.device_guard(dev):
        _native.check(lib.bs_fp8_tp_reduce_switch(
            data_multicast, flags.data_ptr(), flags_multicast, data.numel(), rank, world, epoch, limit_ns,
            _native.stream_handle(dev)), "bs_fp8_tp_reduce_switch")
    return data


def tp_flag_words(world: int) -> int:
    """int32 words of the flag buffer tp_reduce_switch needs for `world` ranks."""
    return int(_native.lib().bs_fp8_tp_flag_words(world))


def gemm_silu_quant(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, *,
                    b_tiled: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """gate_up GEMM + SiLU(gate)*up + per-token-group quant: B holds [gate; up] (2I rows).
    Returns Q e4m3 [..., I] and Qs fp32 [..., I/128]."""
    dev, A2, As2, Bs2, M, N2, K = _check_operands(A, B, As, Bs, b_tiled)
    _need(N2 % (2 * BLOCK) == 0, "gate_up rows must be a multiple of 256")
    inter = N2 // 2
    Q = torch.empty((*A.shape[:-1], inter), dtype=E4M3, device=dev)
    Qs = torch.empty((*A.shape[:-1], inter // BLOCK), dtype=torch.float32, device=dev)
    lib = _native.lib()
    with _native.device_guard(dev):
        ws_bytes = lib.bs_fp8_workspace_bytes(M, N2, K, 1)
        ws = _native.workspace(dev, ws_bytes)
        _native.check(lib.bs_fp8_gemm_silu_quant(
            A2.data_ptr(), _as_bytes(B).data_ptr(), Q.data_ptr(), As2.data_ptr(), Bs2.data_ptr(), Qs.data_ptr(),
            M, N2, K, int(b_tiled), _native.ptr(ws), 0 if ws is None else ws.numel(),
            _native.stream_handle(dev)), "bs_fp8_gemm_silu_quant")
    return Q, Qs


# ------------------------------------------------------------------ mixture of experts
@dataclass(slots=True)
class MoeRoute:
    """A routed batch of T tokens with k slots each (moe_route, moe_dispatch), all on the device. Rows are the
    (token, slot) pairs whose expert is local, sorted by expert and then by place in ids.

      weights    fp32 [T, k]           weight of each slot
      ids        int32 [T, k]          expert of each slot, -1 for none
      offsets    int32 [experts + 1]   rows of local expert e: offsets[e] .. offsets[e + 1] - 1
      row_token  int32 [T * k]         token of each row, -1 past offsets[-1]
      slot_row   int32 [T, k]          row of each slot, -1 when its expert is not local
      num_experts  experts in all (None: the local ones)
    """
    weights: torch.Tensor | None
    ids: torch.Tensor
    offsets: torch.Tensor
    row_token: torch.Tensor
    slot_row: torch.Tensor
    num_experts: int | None = None


def _local_experts(experts, num_experts: int) -> tuple[int, int]:
    begin, count = (0, num_experts) if experts is None else experts
    _need(0 <= begin and 0 < count and begin + count <= num_experts, "experts must be a (begin, count) range of them")
    return begin, count


def _plan_buffers(T: int, k: int, count: int, dev: torch.device, with_ids: bool):
    """One allocation: [weights | ids |] row_token | slot_row | offsets | scratch, in int32 words."""
    R = T * k
    scratch = _native.lib().bs_fp8_moe_scratch_bytes(T, count) // 4
    head = 2 * R if with_ids else 0
    buf = torch.empty(head + 2 * R + count + 1 + scratch, dtype=torch.int32, device=dev)
    row_token, slot_row = buf[head:head + R], buf[head + R:head + 2 * R].view(T, k)
    at = head + 2 * R
    return buf, row_token, slot_row, buf[at:at + count + 1], buf.data_ptr() + 4 * (at + count + 1), 4 * scratch


def moe_route(logits: torch.Tensor, top_k: int, *, renormalize: bool = True, scale: float = 1.0,
              experts: tuple[int, int] | None = None) -> MoeRoute:
    """Router of a mixture of experts: logits [T, E] (bf16 or fp32) -> the top_k experts of each token (largest
    logits, equal ones by lower index), their weights scale * softmax (over the chosen, or over all experts with
    renormalize=False), and the dispatch plan for the local experts (begin, count) (None: all). Logits of -inf
    or NaN are never chosen; slots left over have id -1 and weight 0."""
    _need(logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32), "logits must be bf16 or fp32 [T, E]")
    dev = _cuda(logits)
    T, E = logits.shape
    _need(0 < E <= MAX_EXPERTS, f"1 to {MAX_EXPERTS} experts are supported")
    _need(0 < top_k <= min(E, MAX_TOP_K), f"top_k must be 1 to {MAX_TOP_K} and at most the number of experts")
    begin, count = _local_experts(experts, E)
    if logits.stride(1) != 1 or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    with _native.device_guard(dev):
        buf, row_token, slot_row, offsets, scratch, scratch_bytes = _plan_buffers(T, top_k, count, dev, True)
        R = T * top_k
        weights, ids = buf[:R].view(torch.float32).view(T, top_k), buf[R:2 * R].view(T, top_k)
        base = buf.data_ptr()
        _native.check(_native.lib().bs_fp8_moe_route(
            logits.data_ptr(), int(logits.dtype == torch.float32), max(E, logits.stride(0)), T, E, top_k,
            int(renormalize), float(scale), begin, count, base, base + 4 * R, offsets.data_ptr(), base + 8 * R,
            base + 12 * R, scratch, scratch_bytes, _native.stream_handle(dev)), "bs_fp8_moe_route")
    return MoeRoute(weights, ids, offsets, row_token, slot_row, E)


def moe_dispatch(ids: torch.Tensor, weights: torch.Tensor | None, num_experts: int, *,
                 experts: tuple[int, int] | None = None) -> MoeRoute:
    """The dispatch plan of a routing made elsewhere: ids int32 [T, k] (an id outside the local experts, such as
    -1, has no row), weights fp32 [T, k] (None if no weighted sum follows)."""
    _need(ids.dim() == 2 and ids.dtype == torch.int32, "ids must be int32 [T, k]")
    dev = _cuda(ids) if weights is None else _cuda(ids, weights)
    _need(weights is None or (weights.dtype == torch.float32 and weights.shape == ids.shape), "weights must be fp32 like ids")
    T, k = ids.shape
    _need(0 < num_experts <= MAX_EXPERTS, f"1 to {MAX_EXPERTS} experts are supported")
    _need(0 < k <= MAX_TOP_K, f"1 to {MAX_TOP_K} slots per token are supported")
    begin, count = _local_experts(experts, num_experts)
    ids = ids.contiguous()
    with _native.device_guard(dev):
        buf, row_token, slot_row, offsets, scratch, scratch_bytes = _plan_buffers(T, k, count, dev, False)
        _native.check(_native.lib().bs_fp8_moe_dispatch(
            ids.data_ptr(), T, num_experts, k, begin, count, offsets.data_ptr(), row_token.data_ptr(),
            slot_row.data_ptr(), scratch, scratch_bytes, _native.stream_handle(dev)), "bs_fp8_moe_dispatch")
    return MoeRoute(None if weights is None else weights.contiguous(), ids, offsets, row_token, slot_row, num_experts)


def _check_grouped(A, B, As, Bs, route: MoeRoute, b_tiled: bool):
    """Checks and geometry of a grouped product: (device, A, As, Bs, rows of A, R, rows expected, E, N, K)."""
    _need(A.dim() == 2 and A.dtype in (E4M3, torch.uint8), "A must be e4m3 [rows, K]")
    _need(B.dtype in (E4M3, torch.uint8) and B.is_contiguous(), "weights must be contiguous e4m3")
    if b_tiled:
        _need(B.dim() == 5 and tuple(B.shape[3:]) == (BLOCK, BLOCK),
              "tile-first weights must be [E, N/128, K/128, 128, 128] bytes")
        E, N, K = B.shape[0], B.shape[1] * BLOCK, B.shape[2] * BLOCK
    else:
        _need(B.dim() == 3, "row-major weights must be e4m3 [E, N, K]")
        E, N, K = B.shape
        _need(N % BLOCK == 0 and K % BLOCK == 0, "N and K must be multiples of 128")
    off, rt = route.offsets, route.row_token
    dev = _cuda(A, B, As, Bs, off, rt)
    _need(off.dtype == torch.int32 and rt.dtype == torch.int32 and off.is_contiguous() and rt.is_contiguous(),
          "the route's plan must be contiguous int32")
    _need(0 < E <= MAX_EXPERTS and off.shape == (E + 1,), f"the route has {off.numel() - 1} local experts, the weights {E}")
    _need(A.shape[1] == K, f"A has K={A.shape[1]}, weights have K={K}")
    _need(As.dtype == torch.float32 and Bs.dtype == torch.float32, "scales must be fp32")
    _need(As.shape == (A.shape[0], K // BLOCK), "As must be [rows, K/128]")
    _need(Bs.shape == (E, N // BLOCK, K // BLOCK), "Bs must be [E, N/128, K/128]")
    if not A.is_contiguous():
        A = A.contiguous()
    R = rt.numel()
    hint = R if not route.num_experts else -(-R * E // route.num_experts)
    return dev, A, As.contiguous(), Bs.contiguous(), A.shape[0], R, min(hint, R), E, N, K


def grouped_gemm(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, route: MoeRoute, *,
                 b_tiled: bool = False, gather: bool = False, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Block-scaled FP8 product of each row with its expert's weights: C[r] = gemm(A[r], B[e]) for the rows r of
    expert e in `route`, bf16 or fp32 [T * k, N]. A holds the rows themselves (e.g. grouped_gemm_silu_quant's Q), or
    with gather=True the tokens. Rows past route.offsets[-1] are not written."""
    dev, A, As, Bs, rows_a, R, hint, E, N, K = _check_grouped(A, B, As, Bs, route, b_tiled)
    _need(gather or rows_a >= R, f"A has {rows_a} rows, the route has {R}")
    if out is None:
        out = torch.empty((R, N), dtype=out_dtype, device=dev)
    _need(out.dtype in (torch.bfloat16, torch.float32), "output must be bf16 or fp32")
    _need(out.device == dev and out.shape == (R, N) and out.stride(1) == 1, "output must be [T * k, N] with contiguous rows")
    with _native.device_guard(dev):
        _native.check(_native.lib().bs_fp8_grouped_gemm(
            A.data_ptr(), B.data_ptr(), out.data_ptr(), As.data_ptr(), Bs.data_ptr(), route.offsets.data_ptr(),
            route.row_token.data_ptr() if gather else None, rows_a, R, hint, E, N, K, out.stride(0) if R > 1 else N,
            int(b_tiled), int(out.dtype == torch.float32), _native.stream_handle(dev)), "bs_fp8_grouped_gemm")
    return out


def grouped_gemm_silu_quant(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, route: MoeRoute, *,
                            b_tiled: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """gemm_silu_quant of each row's token with its expert's [gate; up] weights: A e4m3 [T, K] holds the tokens, read
    in place through route.row_token. Returns Q e4m3 [T * k, I] and Qs fp32 [T * k, I/128] in row order; rows
    past route.offsets[-1] are not written."""
    dev, A, As, Bs, rows_a, R, hint, E, N2, K = _check_grouped(A, B, As, Bs, route, b_tiled)
    _need(N2 % (2 * BLOCK) == 0, "gate_up rows must be a multiple of 256")
    inter = N2 // 2
    Q = torch.empty((R, inter), dtype=E4M3, device=dev)
    Qs = torch.empty((R, inter // BLOCK), dtype=torch.float32, device=dev)
    with _native.device_guard(dev):
        _native.check(_native.lib().bs_fp8_grouped_gemm_silu_quant(
            A.data_ptr(), B.data_ptr(), Q.data_ptr(), As.data_ptr(), Bs.data_ptr(), Qs.data_ptr(),
            route.offsets.data_ptr(), route.row_token.data_ptr(), rows_a, R, hint, E, N2, K, int(b_tiled),
            _native.stream_handle(dev)), "bs_fp8_grouped_gemm_silu_quant")
    return Q, Qs


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous rows that start on 16 bytes (a copy where they do not)."""
    per16 = 16 // t.element_size()
    if t.stride(-1) != 1 or (t.shape[0] > 1 and (t.stride(0) % per16 or t.stride(0) < t.shape[1])) or t.data_ptr() % 16:
        return t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def block_norm_quant(y: torch.Tensor, residual: torch.Tensor, *, post_weight: torch.Tensor | None = None,
                     gate: torch.Tensor | None = None, scale: float = 1.0, residual_scale: float = 1.0,
                     pre_weight: torch.Tensor | None = None, eps: float = 1e-6, route: MoeRoute | None = None,
                     out: torch.Tensor | None = None):
    """The end of a block and the start of the next one, in one pass and in fp32:
      z = y, or with `route` the experts' rows summed per token, sum_s weights[t, s] * y[slot_row[t, s]]
      n = rmsnorm(z) * post_weight                     (post_weight None: n = z)
      h = residual_scale * residual + scale * gate * n
      A, As = group_quant(rmsnorm(h) * pre_weight)     (pre_weight None: not made)
    y bf16 [T, H] (or [rows, H] with `route`), residual bf16 or fp32 [T, H], gate bf16 [H], [T, 1] or [T, H]. h is
    rounded once, into `out` (a new tensor like residual; pass out=residual to update it in place); A is
    taken from the unrounded h. Returns (h, A e4m3 [T, H], As fp32 [T, H/128]), or h alone without pre_weight."""
    bf16 = torch.bfloat16
    _need(y.dim() == 2 and y.dtype == bf16, "y must be bf16 [rows, H]")
    _need(residual.dim() == 2 and residual.dtype in (bf16, torch.float32), "residual must be bf16 or fp32 [T, H]")
    dev = _cuda(y, residual)
    T, H = residual.shape
    _need(H % BLOCK == 0 and 0 < H <= 16384, "H must be a multiple of 128, at most 16384")
    _need(y.shape[1] == H and (route is not None or y.shape[0] == T), "y must have residual's shape (or be a route's rows)")
    y, residual = _rows16(y), _rows16(residual)
    for w in (post_weight, pre_weight):
        _need(w is None or (w.shape == (H,) and w.dtype == bf16 and w.device == dev and w.is_contiguous()
                            and w.data_ptr() % 16 == 0), "norm weights must be contiguous bf16 [H] on the same device")
    kind, ldg = 0, 0
    if gate is not None:
        _need(gate.dtype == bf16 and gate.device == dev, "gate must be bf16 on the same device")
        if gate.dim() == 1:
            _need(gate.shape == (H,), "gate must be [H], [T, 1] or [T, H]")
            kind, gate = 1, gate.contiguous()
            if gate.data_ptr() % 16:
                gate = gate.clone()
        else:
            _need(gate.dim() == 2 and gate.shape[0] == T and gate.shape[1] in (1, H), "gate must be [H], [T, 1] or [T, H]")
            if gate.shape[1] == 1:
                if T > 1 and gate.stride(0) < 1:
                    gate = gate.contiguous()
                kind, ldg = 2, gate.stride(0) if T > 1 else 1
            else:
                gate = _rows16(gate)
                kind, ldg = 3, _row_stride(gate)
    w_ptr = s_ptr = None
    k = 0
    if route is not None:
        _need(route.weights is not None and route.weights.shape == route.slot_row.shape, "the route has no weights")
        _cuda(y, route.weights, route.slot_row)
        _need(route.weights.dtype == torch.float32 and route.weights.is_contiguous()
              and route.slot_row.dtype == torch.int32 and route.slot_row.is_contiguous(),
              "the route's weights and rows must be contiguous fp32 and int32")
        _need(route.slot_row.shape[0] == T, f"the route has {route.slot_row.shape[0]} tokens, the residual {T}")
        w_ptr, s_ptr, k = route.weights.data_ptr(), route.slot_row.data_ptr(), route.slot_row.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=residual.dtype, device=dev)
    _need(out.shape == (T, H) and out.dtype == residual.dtype and out.device == dev and _rows16(out) is out,
          "out must be like residual, with contiguous 16-byte aligned rows")
    A = As = None
    if pre_weight is not None:
        A = torch.empty((T, H), dtype=E4M3, device=dev)
        As = torch.empty((T, H // BLOCK), dtype=torch.float32, device=dev)
    with _native.device_guard(dev):
        _native.check(_native.lib().bs_fp8_block_norm_quant(
            y.data_ptr(), _row_stride(y), y.shape[0], w_ptr, s_ptr, k, residual.data_ptr(), _row_stride(residual),
            out.data_ptr(), _row_stride(out), int(residual.dtype == torch.float32), _native.ptr(post_weight),
            _native.ptr(gate), kind, ldg, float(scale), float(residual_scale), _native.ptr(pre_weight), float(eps),
            _native.ptr(A), _native.ptr(As), T, H, _native.stream_handle(dev)), "bs_fp8_block_norm_quant")
    return out if pre_weight is None else (out, A, As)
