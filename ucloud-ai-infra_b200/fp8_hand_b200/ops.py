"""Tensor-level entry points over the C-ABI: activation quant, weight pre-pack, block-scaled FP8
GEMM and the fused gate_up + SiLU*up + quant front half; for mixtures of experts the router with its
dispatch plan, the products grouped by expert, and the block's end with its norms.

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
MAX_ROWS = 1 << 30  # tokens times slots: rows are 32-bit on the device and in the C-ABI, which would wrap silently
_BYTES = (E4M3, torch.uint8)


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
# At decode sizes the kernels of these operators take a few microseconds, so the checks below are written for the
# host's time: no message is built and no view is made unless it is needed.
@dataclass(slots=True)
class MoeRoute:
    """A routed batch of T tokens with k slots each (moe_route, moe_dispatch), all on the device. Rows are the
    (token, slot) pairs whose expert is local, sorted by expert and then by place in ids.

      weights    fp32 [T, k]           weight of each slot (None: not known)
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


def _one_device(*ts: torch.Tensor) -> int:
    """Index of the CUDA device that holds every tensor."""
    index = ts[0].get_device()
    for t in ts:
        if t.get_device() != index or index < 0:
            _cuda(*ts)
            raise ValueError("all tensors must be on the same CUDA device")
    return index


def _matrix(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)  # a third cheaper than torch.empty


def _local_experts(experts, num_experts: int) -> tuple[int, int]:
    if experts is None:
        return 0, num_experts
    begin, count = experts
    _need(0 <= begin and 0 < count and begin + count <= num_experts, "experts must be a (begin, count) range of them")
    return begin, count


def _routing_limits(T: int, num_experts: int, k: int) -> None:
    _need(0 < num_experts <= MAX_EXPERTS, f"1 to {MAX_EXPERTS} experts are supported")
    _need(0 < k <= MAX_TOP_K, f"1 to {MAX_TOP_K} slots per token are supported")
    _need(T * k <= MAX_ROWS, f"at most {MAX_ROWS} rows (tokens times slots) are supported")


def _offsets_and_scratch(lib, T: int, count: int, device: torch.device):
    """offsets [count + 1], and the address and bytes of the scratch behind it (one allocation)."""
    scratch = lib.bs_fp8_moe_scratch_bytes(T, count)
    if not scratch:
        return torch.empty_strided((count + 1,), (1,), dtype=torch.int32, device=device), None, 0
    buf = torch.empty(count + 1 + scratch // 4, dtype=torch.int32, device=device)
    return buf[:count + 1], buf.data_ptr() + 4 * (count + 1), scratch


def moe_route(logits: torch.Tensor, top_k: int, *, renormalize: bool = True, scale: float = 1.0,
              experts: tuple[int, int] | None = None) -> MoeRoute:
    """Router of a mixture of experts: logits [T, E] (bf16 or fp32) -> the top_k experts of each token (largest
    logits, equal ones by lower index), their weights scale * softmax (over the chosen, or over all experts with
    renormalize=False), and the dispatch plan for the local experts (begin, count) (None: all). Logits of -inf
    or NaN are never chosen; slots left over have id -1 and weight 0."""
    f32 = logits.dtype == torch.float32
    if logits.dim() != 2 or not (f32 or logits.dtype == torch.bfloat16):
        raise ValueError("logits must be bf16 or fp32 [T, E]")
    T, E = logits.shape
    if not (0 < E <= MAX_EXPERTS and 0 < top_k <= MAX_TOP_K and top_k <= E and T * top_k <= MAX_ROWS):
        _routing_limits(T, E, top_k)
        raise ValueError("top_k must be at most the number of experts")
    index = _one_device(logits)
    begin, count = _local_experts(experts, E)
    ld, inner = logits.stride()
    if inner != 1 or ld < E:
        if inner != 1 or T > 1:
            logits = logits.contiguous()
        ld = E
    lib, dev = _native.lib(), logits.device
    weights = _matrix(T, top_k, torch.float32, dev)
    ids, slot_row = _matrix(T, top_k, torch.int32, dev), _matrix(T, top_k, torch.int32, dev)
    row_token = torch.empty_strided((T * top_k,), (1,), dtype=torch.int32, device=dev)
    offsets, scratch, scratch_bytes = _offsets_and_scratch(lib, T, count, dev)
    _native.call(lib.bs_fp8_moe_route, "bs_fp8_moe_route", index, logits.data_ptr(), f32, ld, T, E, top_k, renormalize,
                 scale, begin, count, weights.data_ptr(), ids.data_ptr(), offsets.data_ptr(), row_token.data_ptr(),
                 slot_row.data_ptr(), scratch, scratch_bytes)
    return MoeRoute(weights, ids, offsets, row_token, slot_row, E)


def moe_dispatch(ids: torch.Tensor, weights: torch.Tensor | None, num_experts: int, *,
                 experts: tuple[int, int] | None = None) -> MoeRoute:
    """The dispatch plan of a routing made elsewhere: ids int32 [T, k] (an id outside the local experts, such as
    -1, has no row), weights fp32 [T, k] (None if no weighted sum follows)."""
    if ids.dim() != 2 or ids.dtype != torch.int32:
        raise ValueError("ids must be int32 [T, k]")
    T, k = ids.shape
    if not (0 < num_experts <= MAX_EXPERTS and 0 < k <= MAX_TOP_K and T * k <= MAX_ROWS):
        _routing_limits(T, num_experts, k)
    if weights is not None:
        if weights.dtype != torch.float32 or weights.shape != ids.shape:
            raise ValueError("weights must be fp32 like ids")
        index = _one_device(ids, weights)
        weights = weights.contiguous()
    else:
        index = _one_device(ids)
    begin, count = _local_experts(experts, num_experts)
    ids = ids.contiguous()
    lib, dev = _native.lib(), ids.device
    rows = torch.empty((2, T * k), dtype=torch.int32, device=dev)
    row_token, slot_row = rows[0], rows[1].view(T, k)
    offsets, scratch, scratch_bytes = _offsets_and_scratch(lib, T, count, dev)
    _native.call(lib.bs_fp8_moe_dispatch, "bs_fp8_moe_dispatch", index, ids.data_ptr(), T, num_experts, k, begin, count,
                 offsets.data_ptr(), row_token.data_ptr(), slot_row.data_ptr(), scratch, scratch_bytes)
    return MoeRoute(weights, ids, offsets, row_token, slot_row, num_experts)


def _check_grouped(A, B, As, Bs, route: MoeRoute, b_tiled: bool):
    """Checks and geometry of a grouped product: (device index, A, As, Bs, rows of A, R, rows expected, E, N, K)."""
    off, rt = route.offsets, route.row_token
    index = _one_device(A, B, As, Bs, off, rt)
    if b_tiled:
        if B.dim() != 5:
            raise ValueError("tile-first weights must be [E, N/128, K/128, 128, 128] bytes")
        E, nb, kb, r, c = B.shape
        if r != BLOCK or c != BLOCK:
            raise ValueError("tile-first weights must be [E, N/128, K/128, 128, 128] bytes")
        N, K = nb * BLOCK, kb * BLOCK
    else:
        if B.dim() != 3:
            raise ValueError("row-major weights must be e4m3 [E, N, K]")
        E, N, K = B.shape
        if N % BLOCK or K % BLOCK:
            raise ValueError("N and K must be multiples of 128")
        nb, kb = N // BLOCK, K // BLOCK
    if B.dtype not in _BYTES or not B.is_contiguous():
        raise ValueError("weights must be contiguous e4m3")
    if A.dim() != 2 or A.dtype not in _BYTES:
        raise ValueError("A must be e4m3 [rows, K]")
    rows_a, ka = A.shape
    if ka != K:
        raise ValueError(f"A has K={ka}, weights have K={K}")
    if As.dtype != torch.float32 or Bs.dtype != torch.float32:
        raise ValueError("scales must be fp32")
    if As.shape != (rows_a, kb) or Bs.shape != (E, nb, kb):
        raise ValueError("As must be [rows, K/128] and Bs [E, N/128, K/128]")
    if off.dtype != torch.int32 or rt.dtype != torch.int32 or not (off.is_contiguous() and rt.is_contiguous()):
        raise ValueError("the route's plan must be contiguous int32")
    if not 0 < E <= MAX_EXPERTS or off.numel() != E + 1:
        raise ValueError(f"the route has {off.numel() - 1} local experts, the weights {E} (at most {MAX_EXPERTS})")
    R = rt.numel()
    hint = min(R, -(-R * E // route.num_experts)) if route.num_experts else R
    return index, A.contiguous(), As.contiguous(), Bs.contiguous(), rows_a, R, hint, E, N, K


def grouped_gemm(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, route: MoeRoute, *,
                 b_tiled: bool = False, gather: bool = False, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Block-scaled FP8 product of each row with its expert's weights: C[r] = gemm(A[r], B[e]) for the rows r of
    expert e in `route`, bf16 or fp32 [T * k, N]. A holds the rows themselves (e.g. grouped_gemm_silu_quant's Q), or
    with gather=True the tokens. Rows past route.offsets[-1] are not written."""
    index, A, As, Bs, rows_a, R, hint, E, N, K = _check_grouped(A, B, As, Bs, route, b_tiled)
    need = route.slot_row.shape[0] if gather else R
    if rows_a < need:
        raise ValueError(f"A has {rows_a} rows, the route has {need} {'tokens' if gather else 'rows'}")
    if out is None:
        out, ldc = _matrix(R, N, out_dtype, A.device), N
    else:
        if out.shape != (R, N) or out.get_device() != index or out.stride(1) != 1:
            raise ValueError("output must be [T * k, N] with contiguous rows, on the same device")
        ldc = out.stride(0) if R > 1 else N
        if ldc >= 1 << 31:
            raise ValueError("the output's row stride must be below 2^31 elements")
    f32 = out.dtype == torch.float32
    if not f32 and out.dtype != torch.bfloat16:
        raise ValueError("output must be bf16 or fp32")
    _native.call(_native.lib().bs_fp8_grouped_gemm, "bs_fp8_grouped_gemm", index, A.data_ptr(), B.data_ptr(), out.data_ptr(),
                 As.data_ptr(), Bs.data_ptr(), route.offsets.data_ptr(), route.row_token.data_ptr() if gather else None,
                 rows_a, R, hint, E, N, K, ldc, b_tiled, f32)
    return out


def grouped_gemm_silu_quant(A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, route: MoeRoute, *,
                            b_tiled: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """gemm_silu_quant of each row's token with its expert's [gate; up] weights: A e4m3 [T, K] holds the tokens, read
    in place through route.row_token. Returns Q e4m3 [T * k, I] and Qs fp32 [T * k, I/128] in row order; rows
    past route.offsets[-1] are not written."""
    index, A, As, Bs, rows_a, R, hint, E, N2, K = _check_grouped(A, B, As, Bs, route, b_tiled)
    if rows_a < route.slot_row.shape[0]:
        raise ValueError(f"A has {rows_a} rows, the route has {route.slot_row.shape[0]} tokens")
    if N2 % (2 * BLOCK):
        raise ValueError("gate_up rows must be a multiple of 256")
    dev = A.device
    Q = _matrix(R, N2 // 2, E4M3, dev)
    Qs = _matrix(R, N2 // (2 * BLOCK), torch.float32, dev)
    _native.call(_native.lib().bs_fp8_grouped_gemm_silu_quant, "bs_fp8_grouped_gemm_silu_quant", index, A.data_ptr(),
                 B.data_ptr(), Q.data_ptr(), As.data_ptr(), Bs.data_ptr(), Qs.data_ptr(), route.offsets.data_ptr(),
                 route.row_token.data_ptr(), rows_a, R, hint, E, N2, K, b_tiled)
    return Q, Qs


def _rows16(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(t with contiguous rows that start on 16 bytes, copied where they do not; its row stride)."""
    rows, n = t.shape
    if t.is_contiguous():
        ld = n
    else:
        ld, inner = t.stride()
        if rows <= 1:
            ld = n
        if inner != 1 or ld < n:
            return t.clone(memory_format=torch.contiguous_format), n
    if (ld * t.element_size()) % 16 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format), n
    return t, ld


def _norm_weight(w: torch.Tensor, H: int, index: int) -> int:
    """The address of a norm's weight."""
    at = w.data_ptr()
    if w.dtype != torch.bfloat16 or w.shape != (H,) or w.get_device() != index or at % 16 or not w.is_contiguous():
        raise ValueError("norm weights must be contiguous, 16-byte aligned bf16 [H] on the same device")
    return at


def _gate(gate: torch.Tensor, T: int, H: int, index: int) -> tuple[torch.Tensor, int, int]:
    """(the gate, copied where its rows are not contiguous; its kind in the C-ABI; its row stride)."""
    if gate.dtype != torch.bfloat16 or gate.get_device() != index:
        raise ValueError("gate must be bf16 on the same device")
    if gate.dim() == 1 and gate.shape[0] == H:
        if gate.data_ptr() % 16 or not gate.is_contiguous():
            gate = gate.clone(memory_format=torch.contiguous_format)
        return gate, 1, 0
    if gate.dim() != 2 or gate.shape[0] != T or gate.shape[1] not in (1, H):
        raise ValueError("gate must be [H], [T, 1] or [T, H]")
    if gate.shape[1] == 1:
        ld = gate.stride(0) if T > 1 else 1
        if ld < 1:
            gate, ld = gate.contiguous(), 1
        return gate, 2, ld
    gate, ld = _rows16(gate)
    return gate, 3, ld


def block_norm_quant(y: torch.Tensor, residual: torch.Tensor | None, *, post_weight: torch.Tensor | None = None,
                     gate: torch.Tensor | None = None, scale: float = 1.0, residual_scale: float = 1.0,
                     pre_weight: torch.Tensor | None = None, eps: float = 1e-6, route: MoeRoute | None = None,
                     out: torch.Tensor | None = None, norm_out: bool = False):
    """The end of a block and the start of the next one, in one pass and in fp32:
      z = y, or with `route` the experts' rows summed per token, sum_s weights[t, s] * y[slot_row[t, s]]
      n = rmsnorm(z) * post_weight                     (post_weight None: n = z)
      h = residual_scale * residual + scale * gate * n
      A, As = group_quant(rmsnorm(h) * pre_weight)     (pre_weight None: not made)
    y bf16 [T, H] (or with `route` [T * k, H], or more rows), residual bf16 or fp32 [T, H] (None: h = scale * gate * n, bf16), gate
    bf16 [H], [T, 1] or [T, H]. h is rounded once, into `out` (a new tensor like residual; pass out=residual to update
    it in place); A is taken from the unrounded h. Returns (h, A e4m3 [T, H], As fp32 [T, H/128]), with norm_out also
    the norm itself in bf16 (a router's input), or h alone without pre_weight."""
    bf16 = torch.bfloat16
    if y.dim() != 2 or y.dtype != bf16:
        raise ValueError("y must be bf16 [rows, H]")
    rows_y, hy = y.shape
    index, dev = y.get_device(), y.device
    if residual is None:
        wide, H = False, hy
        T = rows_y if route is None else route.slot_row.shape[0]
    else:
        wide = residual.dtype == torch.float32
        if residual.dim() != 2 or not (wide or residual.dtype == bf16):
            raise ValueError("residual must be bf16 or fp32 [T, H]")
        if index < 0 or residual.get_device() != index:
            _one_device(y, residual)
        T, H = residual.shape
    if index < 0:
        _one_device(y)
    if H % BLOCK or not 0 < H <= 16384:
        raise ValueError("H must be a multiple of 128, at most 16384")
    if hy != H or (route is None and rows_y != T):
        raise ValueError("y must have residual's shape (or be a route's rows)")
    h_type = torch.float32 if wide else bf16
    given = out
    if out is None:
        out, ldo = _matrix(T, H, h_type, dev), H
    else:
        if out.shape != (T, H) or out.dtype != h_type or out.get_device() != index:
            raise ValueError("out must be like residual")
        same, ldo = _rows16(out)
        if same is not out:
            raise ValueError("out must have contiguous 16-byte aligned rows")
    y, ldy = _rows16(y)
    r_ptr, ldr = None, 0
    if residual is not None:
        residual, ldr = (out, ldo) if residual is given else _rows16(residual)
        r_ptr = residual.data_ptr()
    post = None if post_weight is None else _norm_weight(post_weight, H, index)
    kind, ldg, g_ptr = 0, 0, None
    if gate is not None:
        gate, kind, ldg = _gate(gate, T, H, index)
        g_ptr = gate.data_ptr()
    w_ptr = s_ptr = None
    k = 0
    if route is not None:
        w, rows = route.weights, route.slot_row
        if w is None or w.shape != rows.shape or rows.shape[0] != T:
            raise ValueError("the route must have weights, and a token for each row of the residual")
        if rows_y < rows.numel():
            raise ValueError(f"y has {rows_y} rows, the route has {rows.numel()}")
        if w.get_device() != index or rows.get_device() != index:
            _one_device(y, w, rows)
        if w.dtype != torch.float32 or rows.dtype != torch.int32 or not (w.is_contiguous() and rows.is_contiguous()):
            raise ValueError("the route's weights and rows must be contiguous fp32 and int32")
        w_ptr, s_ptr, k = w.data_ptr(), rows.data_ptr(), rows.shape[1]
    if pre_weight is None:
        if norm_out:
            raise ValueError("norm_out needs pre_weight")
        A = As = V = pre = a_ptr = as_ptr = v_ptr = None
    else:
        pre = _norm_weight(pre_weight, H, index)
        A, As = _matrix(T, H, E4M3, dev), _matrix(T, H // BLOCK, torch.float32, dev)
        V = _matrix(T, H, bf16, dev) if norm_out else None
        a_ptr, as_ptr, v_ptr = A.data_ptr(), As.data_ptr(), _native.ptr(V)
    _native.call(_native.lib().bs_fp8_block_norm_quant, "bs_fp8_block_norm_quant", index, y.data_ptr(), ldy, rows_y, w_ptr,
                 s_ptr, k, r_ptr, ldr, out.data_ptr(), ldo, wide, post, g_ptr, kind, ldg, scale, residual_scale, pre, eps,
                 a_ptr, as_ptr, v_ptr, T, H)
    if pre_weight is None:
        return out
    return (out, A, As, V) if norm_out else (out, A, As)
