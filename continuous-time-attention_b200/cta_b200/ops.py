"""Functional wrappers over the C ABI: torch tensors in, torch tensors out.

These are the single-launch building blocks used by the reference-compatible
modules (``diffusion_triton``, ``pde_layers``, ``transformers``,
``serving_vllm``, ``sharded``).  They validate shapes, allocate outputs with
torch (the library itself never allocates) and enqueue one kernel on the
current CUDA stream.  Callers handle the identity cases (``steps == 0``,
sequence length < 3) with the reference's aliasing rules before calling here.
"""
from __future__ import annotations

import operator
from typing import Optional, Sequence, Union

import torch
from torch.autograd import forward_ad

from . import _lib

AlphaLike = Union[float, torch.Tensor]


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on CUDA")


def _alpha_args(alphas: Sequence[AlphaLike], steps: int, device: torch.device):
    """Host floats -> (float array, NULL); device scalars -> (NULL, pointer array)."""
    if len(alphas) != steps:
        raise ValueError(f"expected {steps} alpha values, got {len(alphas)}")
    if all(not isinstance(a, torch.Tensor) for a in alphas):
        return _lib.float_array(alphas), None, 0, []
    tens = []
    for a in alphas:
        if not isinstance(a, torch.Tensor):
            a = torch.tensor([float(a)], dtype=torch.float32, device=device)
        if a.device != device:
            raise ValueError(f"alpha on {a.device}, expected {device}")
        if a.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            a = a.float()
        if a.numel() < 1:
            raise ValueError("alpha tensor is empty")
        a = a.detach()
        if not a.is_contiguous():
            a = a.contiguous()
        tens.append(a)
    code = _lib.dtype_code(tens[0].dtype)
    if any(t.dtype != tens[0].dtype for t in tens):
        tens = [t.float() for t in tens]
        code = 0
    return None, _lib.ptr_array(tens), code, tens  # keep tensors alive for the call


def _mask_args(mask: Optional[torch.Tensor], B: int, L: int, device: torch.device):
    if mask is None:
        return None, 0, 0, 0
    if mask.dim() != 2 or mask.shape[0] != B or mask.shape[1] != L:
        raise ValueError(f"attention_mask must be ({B}, {L}), got {tuple(mask.shape)}")
    if mask.device != device:
        raise ValueError(f"attention_mask on {mask.device}, expected {device}")
    if mask.dtype == torch.bool:
        mask = mask.view(torch.uint8)
    return mask, _lib.mask_code(mask.dtype), mask.stride(0), mask.stride(1)


def _out(out: Optional[torch.Tensor], shape, like: torch.Tensor, contiguous: bool = False) -> torch.Tensor:
    """The caller's output buffer after checking it, or a new one."""
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"out must be {tuple(shape)} {like.dtype} on {like.device}")
    if out.stride(-1) != 1 or (contiguous and not out.is_contiguous()):
        raise ValueError("out must have a contiguous last axis" + (" and be contiguous" if contiguous else ""))
    return out


def _residual_view(residual: torch.Tensor, shape, like: torch.Tensor) -> torch.Tensor:
    if tuple(residual.shape) != tuple(shape) or residual.dtype != like.dtype or residual.device != like.device:
        raise ValueError(f"residual must be {tuple(shape)} {like.dtype} on {like.device}")
    return residual if residual.stride(-1) == 1 else residual.contiguous()


# ---------------------------------------------------------------------------
# [B, D, L]
# ---------------------------------------------------------------------------
def bdl(
    x: torch.Tensor,
    alphas: Sequence[AlphaLike],
    steps: int,
    *,
    causal: bool = False,
    backward: bool = False,
    mask: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    arith: Optional[str] = None,
) -> torch.Tensor:
    """`steps` fused steps (or their adjoint) on a contiguous [B, D, L] tensor.

    `arith` ("exact" / "contracted", None = the process default) selects the
    forward update's arithmetic for 16-bit tensors (cta_b200.set_arithmetic)."""
    _require_cuda(x, "x")
    if x.dim() != 3:
        raise ValueError("x must have shape (B, D, L)")
    if x.stride(2) != 1 or x.stride(0) != x.shape[1] * x.stride(1):
        x = x.contiguous()
    B, D, L = x.shape
    y = _out(out, x.shape, x, contiguous=True)
    fa, pa, pcode, keep = _alpha_args(alphas, steps, x.device)
    m, mcode, msb, msl = _mask_args(mask, B, L, x.device)
    lib = _lib.load()
    with _lib.on_device(x), _lib.thread_arithmetic(arith):
        rc = lib.cta_diffusion_bdl_ex(
            _lib.ptr(x), _lib.ptr(y), B, D, L, x.stride(1), y.stride(1), _lib.dtype_code(x.dtype), steps,
            int(causal), int(backward), fa, pa, pcode, _lib.ptr(m), mcode, msb, msl, _lib.stream_ptr(x),
        )
    del keep
    _lib.check(rc)
    return y


def bdl_simple(x: torch.Tensor, alpha: float, steps: int, backward: bool = False,
               out: Optional[torch.Tensor] = None, arith: Optional[str] = None) -> torch.Tensor:
    """Reference kernel API path: one host alpha, no mask, non-causal."""
    _require_cuda(x, "x")
    if not x.is_contiguous():
        x = x.contiguous()
    B, D, L = x.shape
    y = _out(out, x.shape, x, contiguous=True)
    lib = _lib.load()
    fn = lib.cta_diffusion_bwd_bdl if backward else lib.cta_diffusion_fwd_bdl
    with _lib.on_device(x), _lib.thread_arithmetic(arith):
        rc = fn(_lib.ptr(x), _lib.ptr(y), B, D, L, L, _lib.dtype_code(x.dtype), steps, float(alpha),
                _lib.stream_ptr(x))
    _lib.check(rc)
    return y


# ---------------------------------------------------------------------------
# [B, L, D]
# ---------------------------------------------------------------------------
def _bld_view(x: torch.Tensor) -> torch.Tensor:
    if x.stride(2) != 1:
        x = x.contiguous()
    return x


def bld_forward(
    x: torch.Tensor,
    alphas: Sequence[AlphaLike],
    steps: int,
    *,
    causal: bool = False,
    mask: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    arith: Optional[str] = None,
) -> torch.Tensor:
    """`steps` fused steps on [B, L, D] (feature axis contiguous), one launch.

    With `residual` (non-causal, host alphas) the same launch returns
    residual + stencil(x), equal bit for bit to the two-pass result.  `arith`
    ("exact" / "contracted", None = the process default) selects the update's
    arithmetic for 16-bit tensors (cta_b200.set_arithmetic)."""
    _require_cuda(x, "x")
    if x.dim() != 3:
        raise ValueError("x must have shape (B, L, D)")
    x = _bld_view(x)
    B, L, D = x.shape
    y = _out(out, (B, L, D), x)
    fa, pa, pcode, keep = _alpha_args(alphas, steps, x.device)
    m, mcode, msb, msl = _mask_args(mask, B, L, x.device)
    lib = _lib.load()
    if residual is not None:
        r = _residual_view(residual, (B, L, D), x)
        if causal or pa is not None:
            raise ValueError("the fused residual add takes the non-causal stencil with host alphas")
        with _lib.on_device(x), _lib.thread_arithmetic(arith):
            rc = lib.cta_diffusion_fwd_bld_residual(
                _lib.ptr(x), _lib.ptr(r), _lib.ptr(y), B, L, D, x.stride(0), x.stride(1), r.stride(0), r.stride(1),
                y.stride(0), y.stride(1), _lib.dtype_code(x.dtype), steps, fa, _lib.ptr(m), mcode, msb, msl,
                _lib.stream_ptr(x),
            )
        del keep
        _lib.check(rc)
        return y
    with _lib.on_device(x), _lib.thread_arithmetic(arith):
        rc = lib.cta_diffusion_fwd_bld(
            _lib.ptr(x), _lib.ptr(y), B, L, D, x.stride(0), x.stride(1), y.stride(0), y.stride(1),
            _lib.dtype_code(x.dtype), steps, int(causal), fa, pa, pcode, _lib.ptr(m), mcode, msb, msl,
            _lib.stream_ptr(x),
        )
    del keep
    _lib.check(rc)
    return y


_WS: "OrderedDict" = None  # (device, stream, tag) -> buffer, most recently used last
_WS_PER_DEVICE = 8


def _workspace(device: torch.device, nbytes: int, tag: str = "dalpha") -> torch.Tensor:
    """Zero-initialised scratch, one per (device, stream, tag), at most
    _WS_PER_DEVICE per device (least recently used dropped first).

    "dalpha": the d(alpha) reductions; their kernels leave the completion
    counters at zero, so the buffer stays reusable without clearing between
    calls on the same stream.  Other users take their own tag, so that nothing
    else ever writes into those counters.  A buffer is only ever used on the
    stream it was allocated on, so dropping it hands its memory back to torch's
    stream-ordered caching allocator without a race against kernels in flight.
    """
    global _WS
    if _WS is None:
        from collections import OrderedDict

        _WS = OrderedDict()
    key = (device, torch.cuda.current_stream(device).cuda_stream, tag)
    buf = _WS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 4096), dtype=torch.uint8, device=device)
        _WS[key] = buf
        same = [k for k in _WS if k[0] == device]
        for k in same[: max(0, len(same) - _WS_PER_DEVICE)]:
            del _WS[k]
    _WS.move_to_end(key)
    return buf


def bld_backward(
    grad_out: torch.Tensor,
    alphas: Sequence[AlphaLike],
    steps: int,
    *,
    x: Optional[torch.Tensor] = None,
    causal: bool = False,
    mask: Optional[torch.Tensor] = None,
    need_dalpha: bool = False,
    out: Optional[torch.Tensor] = None,
    arith: Optional[str] = None,
):
    """grad_in = A_1^T .. A_S^T grad_out; with need_dalpha also d(alpha_k) (fp32 [steps]).
    `arith` as for bld_forward (16-bit tensors; None = the process default)."""
    _require_cuda(grad_out, "grad_out")
    g = _bld_view(grad_out)
    B, L, D = g.shape
    dx = _out(out, (B, L, D), g)
    fa, pa, pcode, keep = _alpha_args(alphas, steps, g.device)
    m, mcode, msb, msl = _mask_args(mask, B, L, g.device)
    lib = _lib.load()
    dalpha = None
    ws = None
    ws_bytes = 0
    xs = None
    if need_dalpha:
        if x is None:
            raise ValueError("need_dalpha requires the forward input x")
        xs = _bld_view(x)
        if xs.dtype != g.dtype or tuple(xs.shape) != (B, L, D):
            raise ValueError("x must match grad_out in shape and dtype")
        dalpha = torch.empty(steps, dtype=torch.float32, device=g.device)
        ws_bytes = int(lib.cta_diffusion_bwd_bld_workspace_bytes(B, L, D, _lib.dtype_code(g.dtype), steps,
                                                                 int(causal)))
        ws = _workspace(g.device, ws_bytes)
    with _lib.on_device(g), _lib.thread_arithmetic(arith):
        rc = lib.cta_diffusion_bwd_bld(
            _lib.ptr(g), _lib.ptr(dx), _lib.ptr(xs), _lib.ptr(dalpha), _lib.ptr(ws), ws_bytes, B, L, D,
            g.stride(0), g.stride(1), xs.stride(0) if xs is not None else 0, xs.stride(1) if xs is not None else 0,
            dx.stride(0), dx.stride(1), _lib.dtype_code(g.dtype), steps, int(causal), fa, pa, pcode, _lib.ptr(m),
            mcode, msb, msl, _lib.stream_ptr(g),
        )
    del keep
    _lib.check(rc)
    return dx, dalpha


def varlen_forward(
    x: torch.Tensor,
    cu_seqlens: torch.Tensor,
    max_len: int,
    alpha: float,
    steps: int,
    *,
    pad_to_max: bool,
    out: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    arith: Optional[str] = None,
) -> torch.Tensor:
    """Packed [T, D] prefill with device cu_seqlens (int32, nseq+1); one launch."""
    _require_cuda(x, "x")
    if x.dim() != 2:
        raise ValueError("x must have shape (T, D)")
    if x.stride(1) != 1:
        x = x.contiguous()
    if cu_seqlens.device != x.device:
        raise ValueError("cu_seqlens must be on the same device as x")
    if cu_seqlens.dtype != torch.int32:
        cu_seqlens = cu_seqlens.to(torch.int32)
    if not cu_seqlens.is_contiguous():
        cu_seqlens = cu_seqlens.contiguous()
    T, D = x.shape
    y = _out(out, (T, D), x, contiguous=True)
    nseq = cu_seqlens.numel() - 1
    lib = _lib.load()
    if residual is not None:
        r = _residual_view(residual, (T, D), x)
        with _lib.on_device(x), _lib.thread_arithmetic(arith):
            rc = lib.cta_diffusion_fwd_varlen_residual(
                _lib.ptr(x), _lib.ptr(r), _lib.ptr(y), T, D, x.stride(0), r.stride(0), y.stride(0),
                _lib.ptr(cu_seqlens), nseq, int(max_len), int(pad_to_max), _lib.dtype_code(x.dtype), steps,
                float(alpha), _lib.stream_ptr(x),
            )
        _lib.check(rc)
        return y
    with _lib.on_device(x), _lib.thread_arithmetic(arith):
        rc = lib.cta_diffusion_fwd_varlen(
            _lib.ptr(x), _lib.ptr(y), T, D, x.stride(0), y.stride(0), _lib.ptr(cu_seqlens), nseq, int(max_len),
            int(pad_to_max), _lib.dtype_code(x.dtype), steps, float(alpha), _lib.stream_ptr(x),
        )
    _lib.check(rc)
    return y


def shard_part(
    x_local: torch.Tensor,
    out: torch.Tensor,
    part: int,
    *,
    pos_offset: int,
    global_len: int,
    alpha: float,
    steps: int,
    causal: bool = False,
    backward: bool = False,
    lo_halo: Optional[torch.Tensor] = None,
    hi_halo: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
    arith: Optional[str] = None,
) -> None:
    """One launch over a part (interior / lo edge / hi edge) of an L-shard."""
    B, Lloc, D = x_local.shape
    for h in (lo_halo, hi_halo):
        if h is not None and (not h.is_contiguous() or h.shape[0] != B or h.shape[2] != D or h.dtype != x_local.dtype):
            raise ValueError("halo must be a contiguous (B, rows, D) tensor of the shard's dtype")
    lo_rows = lo_halo.shape[1] if lo_halo is not None else 0
    hi_rows = hi_halo.shape[1] if hi_halo is not None else 0
    st = stream if stream is not None else torch.cuda.current_stream(x_local.device)
    lib = _lib.load()
    with _lib.on_device(x_local), _lib.thread_arithmetic(arith):
        rc = lib.cta_diffusion_shard_bld(
            _lib.ptr(x_local), _lib.ptr(out), B, Lloc, D, int(pos_offset), int(global_len), _lib.ptr(lo_halo),
            lo_rows, _lib.ptr(hi_halo), hi_rows, int(part), _lib.dtype_code(x_local.dtype), steps, int(causal),
            int(backward), float(alpha), st.cuda_stream,
        )
    _lib.check(rc)


def shard_part_dalpha(
    g_local: torch.Tensor,
    x_local: torch.Tensor,
    dx_out: torch.Tensor,
    dalpha: torch.Tensor,
    part: int,
    *,
    pos_offset: int,
    global_len: int,
    alphas: Sequence[float],
    steps: int,
    causal: bool = False,
    g_lo: Optional[torch.Tensor] = None,
    g_hi: Optional[torch.Tensor] = None,
    x_lo: Optional[torch.Tensor] = None,
    x_hi: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
    arith: Optional[str] = None,
) -> None:
    """One launch over a part of an L-shard's backward with d(alpha): writes the
    part's rows of dx_out and ADDS the part's d(alpha) sum to `dalpha` (fp32 [steps])."""
    B, Lloc, D = g_local.shape
    if tuple(x_local.shape) != (B, Lloc, D) or x_local.dtype != g_local.dtype:
        raise ValueError("x_local must match g_local in shape and dtype")
    if dalpha.dtype != torch.float32 or dalpha.numel() < steps or not dalpha.is_contiguous():
        raise ValueError("dalpha must be a contiguous fp32 tensor of at least `steps` entries")
    for h in (g_lo, g_hi, x_lo, x_hi):
        if h is not None and (not h.is_contiguous() or h.shape[0] != B or h.shape[2] != D or h.dtype != g_local.dtype):
            raise ValueError("halo must be a contiguous (B, rows, D) tensor of the shard's dtype")
    rows = [h.shape[1] if h is not None else 0 for h in (g_lo, g_hi, x_lo, x_hi)]
    if len(alphas) != steps:
        raise ValueError("need one alpha per step")
    st = stream if stream is not None else torch.cuda.current_stream(g_local.device)
    lib = _lib.load()
    code = _lib.dtype_code(g_local.dtype)
    ws_bytes = int(lib.cta_diffusion_bwd_bld_workspace_bytes(B, Lloc, D, code, steps, int(causal)))
    with torch.cuda.stream(st):
        ws = _workspace(g_local.device, ws_bytes)
    with _lib.on_device(g_local), _lib.thread_arithmetic(arith):
        rc = lib.cta_diffusion_shard_bld_dalpha(
            _lib.ptr(g_local), _lib.ptr(x_local), _lib.ptr(dx_out), _lib.ptr(dalpha), _lib.ptr(ws), ws_bytes, B, Lloc,
            D, int(pos_offset), int(global_len), _lib.ptr(g_lo), rows[0], _lib.ptr(g_hi), rows[1], _lib.ptr(x_lo),
            rows[2], _lib.ptr(x_hi), rows[3], int(part), code, steps, int(causal),
            _lib.float_array([float(a) for a in alphas]), st.cuda_stream,
        )
    _lib.check(rc)


def pde_step(
    x: torch.Tensor,
    kind: int,
    alpha: torch.Tensor,
    beta: torch.Tensor,
    *,
    causal: bool = False,
    mask: Optional[torch.Tensor] = None,
    grad_out: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
):
    """One advection- / reaction-diffusion step on [B, L, D] (kind _lib.PDE_*).

    Forward (grad_out None): returns y.  Backward: returns (dx, dcoef) with
    dcoef = fp32 [d(alpha), d(beta)].  alpha, beta: the layer's [1] parameters,
    read on the device."""
    _require_cuda(x, "x")
    if x.dim() != 3:
        raise ValueError("x must have shape (B, L, D)")
    x = _bld_view(x)
    B, L, D = x.shape
    coefs = []
    for c in (alpha, beta):
        c = c.detach()
        if c.device != x.device:
            raise ValueError(f"coefficient on {c.device}, expected {x.device}")
        if c.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            c = c.float()
        coefs.append(c.contiguous())
    if coefs[0].dtype != coefs[1].dtype:
        coefs = [c.float() for c in coefs]
    m, mcode, msb, msl = _mask_args(mask, B, L, x.device)
    lib = _lib.load()
    code = _lib.dtype_code(x.dtype)
    y = _out(out, (B, L, D), x)
    g = None
    dcoef = ws = None
    ws_bytes = 0
    if grad_out is not None:
        g = _bld_view(grad_out)
        if tuple(g.shape) != (B, L, D) or g.dtype != x.dtype:
            raise ValueError("grad_out must match x in shape and dtype")
        dcoef = torch.empty(2, dtype=torch.float32, device=x.device)
        ws_bytes = int(lib.cta_pde_step_workspace_bytes(B, L, D))
        ws = _workspace(x.device, ws_bytes, tag="pde_step")
    with _lib.on_device(x):
        rc = lib.cta_pde_step_bld(
            _lib.ptr(x), _lib.ptr(g), _lib.ptr(y), _lib.ptr(dcoef), _lib.ptr(ws), ws_bytes, B, L, D, x.stride(0),
            x.stride(1), g.stride(0) if g is not None else 0, g.stride(1) if g is not None else 0, y.stride(0),
            y.stride(1), code, int(kind), int(causal), int(grad_out is not None), _lib.ptr(coefs[0]),
            _lib.ptr(coefs[1]), _lib.dtype_code(coefs[0].dtype), _lib.ptr(m), mcode, msb, msl, _lib.stream_ptr(x),
        )
    _lib.check(rc)
    return y if grad_out is None else (y, dcoef)


def pde_stack(
    x: torch.Tensor,
    kind: int,
    alphas: Sequence[torch.Tensor],
    betas: Sequence[torch.Tensor],
    *,
    causal: bool = False,
    mask: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Forward of up to 4 consecutive advection- / reaction-diffusion layers of
    one kind (_lib.PDE_*) on [B, L, D] in one launch, fp32 kept between them.
    alphas[k], betas[k]: layer k's [1] parameters, read on the device."""
    _require_cuda(x, "x")
    if x.dim() != 3:
        raise ValueError("x must have shape (B, L, D)")
    steps = len(alphas)
    if steps != len(betas) or not 1 <= steps <= _lib.PDE_STACK_MAX_STEPS:
        raise ValueError(f"need 1..{_lib.PDE_STACK_MAX_STEPS} alpha / beta pairs")
    x = _bld_view(x)
    B, L, D = x.shape
    coefs = []
    for c in list(alphas) + list(betas):
        c = c.detach()
        if c.device != x.device:
            raise ValueError(f"coefficient on {c.device}, expected {x.device}")
        coefs.append(c.float().contiguous() if c.dtype != torch.float32 else c.contiguous())
    m, mcode, msb, msl = _mask_args(mask, B, L, x.device)
    y = _out(out, (B, L, D), x)
    lib = _lib.load()
    with _lib.on_device(x):
        rc = lib.cta_pde_stack_bld(
            _lib.ptr(x), _lib.ptr(y), B, L, D, x.stride(0), x.stride(1), y.stride(0), y.stride(1),
            _lib.dtype_code(x.dtype), int(kind), steps, int(causal), _lib.ptr_array(coefs[:steps]),
            _lib.ptr_array(coefs[steps:]), 0, _lib.ptr(m), mcode, msb, msl, _lib.stream_ptr(x),
        )
    del coefs
    _lib.check(rc)
    return y


def bld_forward_pool(
    x: torch.Tensor, alphas: Sequence[AlphaLike], steps: int, mask: torch.Tensor
) -> torch.Tensor:
    """`steps` fused non-causal steps on [B, L, D] under `mask`, followed by the
    masked mean pool over L, without writing the stepped tensor: [B, D]."""
    _require_cuda(x, "x")
    if x.dim() != 3:
        raise ValueError("x must have shape (B, L, D)")
    x = _bld_view(x)
    B, L, D = x.shape
    fa, pa, pcode, keep = _alpha_args(alphas, steps, x.device)
    m, mcode, msb, msl = _mask_args(mask, B, L, x.device)
    if m is None:
        raise ValueError("the masked pool needs an attention mask")
    lib = _lib.load()
    pooled = torch.empty((B, D), dtype=x.dtype, device=x.device)
    ws_bytes = int(lib.cta_diffusion_fwd_bld_pool_workspace_bytes(B, L, D))
    ws = _workspace(x.device, ws_bytes, tag="pool")
    with _lib.on_device(x):
        rc = lib.cta_diffusion_fwd_bld_pool(
            _lib.ptr(x), _lib.ptr(pooled), _lib.ptr(ws), ws_bytes, B, L, D, x.stride(0), x.stride(1),
            _lib.dtype_code(x.dtype), steps, fa, pa, pcode, _lib.ptr(m), mcode, msb, msl, _lib.stream_ptr(x),
        )
    del keep
    _lib.check(rc)
    return pooled


# ---------------------------------------------------------------------------
# attention of prompts
# ---------------------------------------------------------------------------
def _same_kind(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")


def _device_ints(t: torch.Tensor, name: str, like: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")
    if t.dtype != dtype:
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
        t = t.to(dtype)
    return t


def _offsets(cu: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    shape = cu.shape
    if len(shape) != 1 or shape[0] < 1:
        raise ValueError("cu_seqlens must have shape (sequences + 1,)")
    if cu.dtype != torch.int32 or cu.get_device() != like.get_device():
        cu = _device_ints(cu, "cu_seqlens", like, torch.int32)
    return cu if cu.is_contiguous() else cu.contiguous()


def _on16(t: torch.Tensor) -> bool:
    """The last axis is contiguous, and every row starts on 16 bytes and on its own."""
    if t.data_ptr() & 15:
        return False
    es = t.element_size()
    if t.is_contiguous():
        return t.shape[-1] * es & 15 == 0  # the other strides are multiples of a row
    s = t.stride()
    return s[-1] == 1 and all(n <= 1 or (x > 0 and x * es & 15 == 0) for x, n in zip(s[:-1], t.shape))


def attention_mask(key_mask: torch.Tensor) -> torch.Tensor:
    """A key mask [B, L] (any mask dtype, non-zero = valid) as the words that
    attention_forward and attention_backward take; one launch."""
    if key_mask.get_device() < 0:
        _require_cuda(key_mask, "key_mask")
    if key_mask.dim() != 2:
        raise ValueError("key_mask must have shape (B, L)")
    B, L = key_mask.shape
    dtype = key_mask.dtype
    code = _lib.mask_code(torch.uint8 if dtype == torch.bool else dtype)  # a bool is a byte
    words = torch.empty((B, _mask_row_words(L)), dtype=torch.int32, device=key_mask.device)
    _lib.enqueue(_lib.load().cta_attention_mask_words, key_mask, key_mask.data_ptr(), code, *key_mask.stride(), B, L,
                 words.data_ptr())
    return words


def _tangents(*tensors: torch.Tensor) -> bool:
    """Whether one carries a forward-mode tangent, which a call would drop.
    Outside of a dual level, a look at its number (unpack_dual takes 0.4 us a tensor)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _attention_inputs(q, k, v, cu_seqlens, mask_words, scale):
    """Checked inputs and sizes: (q, k, v, cu or None, (sequences, length, heads, kv_heads, dim), dtype code, scale)."""
    device = q.get_device()  # plain numbers: comparing device objects costs several times as much
    if device < 0:
        _require_cuda(q, "q")
    dtype = q.dtype
    code = _lib.dtype_code(dtype)
    if k.dtype != dtype or v.dtype != dtype or k.get_device() != device or v.get_device() != device:
        _same_kind(k, "k", q)
        _same_kind(v, "v", q)
    shape, kshape = q.shape, k.shape
    rank = 4 if cu_seqlens is None else 3
    if len(shape) != rank:
        raise ValueError("q must have shape " + ("(B, L, heads, dim)" if rank == 4 else "(T, heads, dim)"))
    if kshape != v.shape or len(kshape) != rank or kshape[:-2] != shape[:-2] or kshape[-1] != shape[-1]:
        raise ValueError(f"q {tuple(shape)}, k {tuple(kshape)}, v {tuple(v.shape)} do not go together")
    length, heads, dim = shape[-3:]
    kv_heads = kshape[-2]
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    cu = None
    if cu_seqlens is None:
        sequences = shape[0]
        if mask_words is not None and (mask_words.dtype != torch.int32 or mask_words.get_device() != device
                                       or not mask_words.is_contiguous()
                                       or mask_words.shape != (sequences, _mask_row_words(length))):
            raise ValueError("mask_words must come from attention_mask() of a (B, L) mask")
    else:
        if mask_words is not None:
            raise ValueError("a key mask takes padded sequences, not packed ones")
        cu = _offsets(cu_seqlens, q)
        sequences = cu.shape[0] - 1
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()
            and (code == 0 or dim & 7 or not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15)):
        q, k, v = _attention_rows(q, code), _attention_rows(k, code), _attention_rows(v, code)
    return q, k, v, cu, (sequences, length, heads, kv_heads, dim), code, dim**-0.5 if scale is None else float(scale)


def _window(window, sinks, causal: bool = True):
    """Checked (window, sinks) as the library takes them, (0, 0) without a window."""
    if window is None:
        if sinks:
            raise ValueError("sinks go with a window")
        return 0, 0
    w, s = operator.index(window), operator.index(sinks)
    if w < 1 or s < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {w} and {s}")
    if not causal:
        raise ValueError("a window needs causal=True")
    return min(w, _FAR), min(s, _FAR)


_FAR = 1 << 40  # more keys than any call has


def _mask_row_words(length: int) -> int:
    """cta_attention_mask_words_per_row: a header of 4 words, then one bit per key in blocks of 128."""
    return 4 + (length + 127) // 128 * 4


def _attention_rows(t: torch.Tensor, code: int) -> torch.Tensor:
    """t with a contiguous last axis and, in 16 bits, rows that the tensor-core kernels can
    load: other views are copied (head dims that are no multiple of 8 take the plain kernels)."""
    if t.stride(-1) == 1 and (code == 0 or t.shape[-1] & 7 or _on16(t)):
        return t
    return _own_rows(t)


def _own_rows(t: torch.Tensor) -> torch.Tensor:
    """A contiguous copy that starts on 16 bytes."""
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _new(like: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of like's shape (empty_like is the cheaper call)."""
    return torch.empty_like(like) if like.is_contiguous() else torch.empty(like.shape, dtype=like.dtype,
                                                                           device=like.device)


def _strides3(t: Optional[torch.Tensor]):
    if t is None:
        return (0, 0, 0)
    s = t.stride()
    return s[:3] if len(s) == 4 else (0, s[0], s[1])


_NO_STRIDES = (0,) * 12


def _low(low: Optional[torch.Tensor], q: torch.Tensor) -> int:
    if low is None:
        return 0
    if (low.shape != q.shape or low.dtype != q.dtype or low.get_device() != q.get_device() or not low.is_contiguous()
            or q.dtype == torch.float32):
        raise ValueError(f"out_low must be contiguous, of a 16-bit type and like q: {tuple(q.shape)}, {q.dtype} on "
                         f"{q.device}")
    return low.data_ptr()


def attention_forward(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    causal: bool = False,
    scale: Optional[float] = None,
    mask_words: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    need_lse: bool = True,
    out_low: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
):
    """Softmax attention of prompts, one launch: (out, lse).

    Padded: q [B, L, heads, dim], k and v [B, L, kv_heads, dim], optionally the
    words of a key mask (attention_mask).  Packed: [T, heads, dim] with device
    cu_seqlens (int32, sequences + 1).  float32, bfloat16, float16; dim up to
    256; any strides (views that TMA cannot address are copied first).  Rows
    that see no key are zero.  Packed rows behind the last sequence keep what
    `out` holds; in an output allocated here they are zero.  `lse` (fp32,
    [B, heads, L] or [heads, T]; None without need_lse) is what
    attention_backward takes.  `out_low`, for 16-bit types a contiguous tensor
    like out, receives what rounding out lost (in float16 times 2048): given to
    attention_backward too, it spares the gradients of rows with few keys the
    error of that rounding.

    `window` (causal only): row i sees the last `window` keys, j > i - window, and the
    first `sinks` ones of its sequence (with a key mask, from its first valid key on);
    what no row of a tile sees costs nothing."""
    reach = _window(window, sinks, causal)
    q, k, v, cu, sizes, code, scale = _attention_inputs(q, k, v, cu_seqlens, mask_words, scale)
    o = _new(q) if out is None else _out(out, q.shape, q)
    return o, _attention_forward(q, k, v, o, _low(out_low, q), cu, mask_words, causal, scale, sizes, code, need_lse,
                                 out is None, reach)


def _attention_forward(q, k, v, o, low, cu, mask_words, causal, scale, sizes, code, need_lse, zero_tail, reach=(0, 0)):
    """attention_forward of inputs that have been checked into o; `low` is an address or 0.  Returns lse."""
    lse = None
    if need_lse:
        n, length, heads = sizes[:3]
        lse = torch.empty((n, heads, length) if cu is None else (heads, length), dtype=torch.float32, device=q.device)
    args = _lib.ATTENTION_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), low, 0 if lse is None else lse.data_ptr(), 0, 0, 0, 0, 0,
        0 if cu is None else cu.data_ptr(), 0 if mask_words is None else mask_words.data_ptr(), *_strides3(q),
        *_strides3(k), *_strides3(v), *_strides3(o), *_NO_STRIDES, *sizes, code, bool(causal), zero_tail, 0, scale, 0.0)
    if reach[0]:
        _lib.enqueue(_lib.load().cta_window_attention_forward, q, args, *reach)
    else:
        _lib.enqueue(_lib.load().cta_attention_forward, q, args)
    return lse


def attention_backward(
    grad_out: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    *,
    causal: bool = False,
    scale: Optional[float] = None,
    mask_words: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    need_dq: bool = True,
    need_dkv: bool = True,
    out_low: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
):
    """(dq, dk, dv) of attention_forward from its out, lse and, if it wrote one, out_low; None for what is not
    wanted."""
    reach = _window(window, sinks, causal)
    q, k, v, cu, sizes, code, scale = _attention_inputs(q, k, v, cu_seqlens, mask_words, scale)
    n, length, heads = sizes[:3]
    if grad_out.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"grad_out and out must be {tuple(q.shape)}")
    device = q.get_device()
    if (grad_out.dtype != q.dtype or out.dtype != q.dtype or grad_out.get_device() != device
            or out.get_device() != device):
        _same_kind(grad_out, "grad_out", q)
        _same_kind(out, "out", q)
    shape = (n, heads, length) if cu is None else (heads, length)
    if lse.shape != shape or lse.dtype != torch.float32 or lse.get_device() != device or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 {shape} on {q.device}")
    return _attention_backward(grad_out, q, k, v, out, _low(out_low, q), lse, cu, mask_words, causal, scale, reach, sizes,
                               code, need_dq, need_dkv)


def _attention_backward(grad_out, q, k, v, out, low, lse, cu, mask_words, causal, scale, reach, sizes, code, need_dq,
                        need_dkv):
    """attention_backward of inputs that have been checked; `low` is an address or 0."""
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()
            and (code == 0 or sizes[4] & 7 or not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15)):
        q, k, v = _attention_rows(q, code), _attention_rows(k, code), _attention_rows(v, code)
    g, o = _attention_rows(grad_out, code), _attention_rows(out, code)
    dq = _new(q) if need_dq else None
    dk = _new(k) if need_dkv else None
    dv = _new(v) if need_dkv else None
    # fp16 on tensor cores: beside delta the norms that scale its score gradients
    planes = 3 if code == 2 else 1
    delta = torch.empty_like(lse) if planes == 1 else torch.empty((planes, *lse.shape), dtype=lse.dtype, device=lse.device)
    args = _lib.ATTENTION_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), low, lse.data_ptr(), g.data_ptr(), delta.data_ptr(),
        _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv), _lib.ptr(cu), _lib.ptr(mask_words), *_strides3(q), *_strides3(k),
        *_strides3(v), *_strides3(o), *_strides3(g), *_strides3(dq), *_strides3(dk), *_strides3(dv), *sizes, code,
        bool(causal), 0, planes, scale, 0.0)
    if not reach[0]:
        _lib.enqueue(_lib.load().cta_attention_backward, q, args)
        return dq, dk, dv
    lib = _lib.load()
    nbytes = _workspace_bytes(lib.cta_window_attention_workspace_bytes, q, args, *reach)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _lib.enqueue(lib.cta_window_attention_backward, q, args, *reach, _lib.ptr(ws), nbytes)
    return dq, dk, dv


def _workspace_bytes(query, t: torch.Tensor, *args) -> int:
    """query(*args) on t's device; raises what the call itself would."""
    if _lib._current_device() == t.get_device():
        nbytes = query(*args)
    else:
        with _lib.on_device(t):
            nbytes = query(*args)
    if nbytes < 0:
        _lib.check(-nbytes)
    return nbytes


# ---------------------------------------------------------------------------
# paged key/value cache
# ---------------------------------------------------------------------------
def _row_strides(t: torch.Tensor):
    """Strides of all axes but the last; an axis of one entry, whose own stride means nothing, counts 0 or
    what it would have in a fresh tensor."""
    if t.is_contiguous():
        shape = t.shape
        if len(shape) == 3:
            return shape[1] * shape[2], shape[2]
        return shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3]
    return tuple(x if n > 1 else 0 for x, n in zip(t.stride(), t.shape[:-1]))


def _placed_rows(t: torch.Tensor):
    """(t or a copy whose rows start on 16 bytes, address, strides of tokens and heads) of rows [T, heads, dim]."""
    address = t.data_ptr()
    if t.is_contiguous() and not address & 15:
        _, heads, dim = t.shape
        if not dim & 7:
            return t, address, heads * dim, dim
    if not _on16(t):
        t = _own_rows(t)
        address = t.data_ptr()
    return (t, address, *_row_strides(t))


def _cache_sizes(k_cache, v_cache, k_scale, v_scale, dtype, like):
    """Checked cache: (pages, page_size, kv_heads, dim, quantized)."""
    shape, kind = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have one shape (pages, page_size, kv_heads, dim)")
    quantized = kind == torch.float8_e4m3fn
    device = like.get_device()
    if (not quantized and kind != dtype) or v_cache.dtype != kind or k_cache.get_device() != device or (
            v_cache.get_device() != device):
        raise ValueError(f"k_cache and v_cache must be {dtype} or float8_e4m3fn on {like.device}, got {kind} on "
                         f"{k_cache.device} and {v_cache.dtype} on {v_cache.device}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and not (k_cache.data_ptr() | v_cache.data_ptr()) & 15
            and shape[3] & 15 == 0) and not (_on16(k_cache) and _on16(v_cache)):
        raise ValueError("k_cache and v_cache must have a contiguous last axis and rows that start on 16 bytes")
    pages, page, heads, dim = shape
    if quantized:
        want = (pages, heads, page)
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if (t is None or t.shape != want or t.dtype != torch.float32 or t.get_device() != device
                    or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous float32 {want} on {like.device}")
    elif k_scale is not None or v_scale is not None:
        raise ValueError("k_scale and v_scale go with a float8_e4m3fn cache")
    return pages, page, heads, dim, quantized


def _slots(slots: torch.Tensor, n: Optional[int], like: torch.Tensor) -> torch.Tensor:
    shape = slots.shape
    if len(shape) != 1 or (n is not None and shape[0] != n):
        raise ValueError("slots must have shape (T,)")
    if slots.dtype != torch.int64 or slots.get_device() != like.get_device():
        slots = _device_ints(slots, "slots", like, torch.int64)
    return slots if slots.is_contiguous() else slots.contiguous()


def _cache_call(fn, k, v, k_cache, v_cache, slots, k_scale, v_scale, sizes):
    pages, page, heads, dim, quantized = sizes
    args = _lib.KV_CACHE_ARGS.pack(
        k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scale), _lib.ptr(v_scale),
        slots.data_ptr(), *_row_strides(k), *_row_strides(v), *_row_strides(k_cache), *_row_strides(v_cache),
        slots.shape[0], heads, dim, pages, page, _lib.dtype_code(k.dtype), quantized)
    _lib.enqueue(fn, k, args)


def kv_cache_write(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    *,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> None:
    """Write rows k, v [T, kv_heads, dim] (bf16 / fp16) into slots [T] (int64) of a paged
    cache [pages, page_size, kv_heads, dim], in place; one launch.

    The cache holds the rows' type, or float8_e4m3fn codes with fp32 scales
    [pages, kv_heads, page_size]: scale = m / 448 and code = e4m3(448 x / m), the
    nearest to the exact quotient, with m = max(max|x|, 2**-100) over the row.  Slot s is entry s % page_size of
    page s // page_size.  A negative slot is skipped (padding rows); the others
    must be distinct.  A slot past the cache is skipped and reported by
    ``_lib.device_error()``."""
    if k.get_device() < 0:
        _require_cuda(k, "k")
    shape = k.shape
    if len(shape) != 3 or shape != v.shape:
        raise ValueError("k and v must have one shape (T, kv_heads, dim)")
    if v.dtype != k.dtype or v.get_device() != k.get_device():
        _same_kind(v, "v", k)
    sizes = _cache_sizes(k_cache, v_cache, k_scale, v_scale, k.dtype, k)
    if shape[1] != sizes[2] or shape[2] != sizes[3]:
        raise ValueError(f"k {tuple(shape)} does not fit a cache {tuple(k_cache.shape)}")
    slots = _slots(slots, shape[0], k)
    k = k if _on16(k) else _own_rows(k)
    v = v if _on16(v) else _own_rows(v)
    _cache_call(_lib.load().cta_kv_cache_write, k, v, k_cache, v_cache, slots, k_scale, v_scale, sizes)


def rotary_cache_write(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    *,
    interleaved: bool = False,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """kv_cache_write of keys that are rotated by their positions on the way; returns the
    queries rotated too.  One launch.

    q [T, heads, dim], k and v [T, kv_heads, dim] (bf16 / fp16), slots [T] and positions [T]
    (int64); the cache as for ``kv_cache_write``.  cos_sin [positions, rotary_dim], float32 or
    q's type, holds the cosines of a position's rotary_dim / 2 angles, then the sines
    (``rotary_table``).  The first rotary_dim elements of a row (a multiple of 16) are
    pairs, elements i and rotary_dim / 2 + i, or with ``interleaved`` 2 i and 2 i + 1;
    pair (a, b) becomes (a cos - b sin, b cos + a sin).  fp32, rounded once; an e4m3 cache
    takes scale and codes from the unrounded row.

    ``out`` receives the queries and may be q itself.  A negative slot leaves the cache
    alone (padding rows; their queries are rotated all the same), the others must be
    distinct.  A slot past the cache is skipped; a token whose position is
    outside of cos_sin has a zero query and is not written.  Both are reported by
    ``_lib.device_error()``, the position only where the slot is not negative.

    Not differentiable: where the queries returned would need a gradient (of q or
    cos_sin) it raises; call it under ``torch.no_grad()`` or on detached tensors.  The
    cache takes no gradients of k and v, as for ``kv_cache_write``."""
    if (torch.is_grad_enabled() and (q.requires_grad or cos_sin.requires_grad)) or _tangents(q, cos_sin):
        raise ValueError("rotary_cache_write has no gradient: q and cos_sin must not require one")
    return _rotary_launch(*_rotary_plan(q, k, v, k_cache, v_cache, slots, positions, cos_sin, interleaved, k_scale,
                                        v_scale, out))


def _rotary_plan(q, k, v, k_cache, v_cache, slots, positions, cos_sin, interleaved, k_scale, v_scale, out):
    """All checks of rotary_cache_write but the library's own, and what its launch takes."""
    device = q.get_device()
    if device < 0:
        _require_cuda(q, "q")
    shape, kshape = q.shape, k.shape
    if len(shape) != 3 or len(kshape) != 3 or kshape != v.shape or kshape[0] != shape[0] or kshape[2] != shape[2]:
        raise ValueError(f"q {tuple(shape)}, k {tuple(kshape)}, v {tuple(v.shape)} must be (T, heads, dim) of one T and dim")
    if k.dtype != q.dtype or v.dtype != q.dtype or k.get_device() != device or v.get_device() != device:
        _same_kind(k, "k", q)
        _same_kind(v, "v", q)
    code = _lib.dtype_code(q.dtype)
    pages, page, kv_heads, dim, quantized = _cache_sizes(k_cache, v_cache, k_scale, v_scale, q.dtype, q)
    if kshape[1] != kv_heads or kshape[2] != dim:
        raise ValueError(f"k {tuple(kshape)} does not fit a cache {tuple(k_cache.shape)}")
    slots = _slots(slots, shape[0], q)
    if positions.dim() != 1 or positions.shape[0] != shape[0]:
        raise ValueError("positions must have shape (T,)")
    if positions.dtype != torch.int64 or positions.get_device() != device:
        positions = _device_ints(positions, "positions", q, torch.int64)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if cos_sin.dim() != 2 or cos_sin.dtype not in (torch.float32, q.dtype) or cos_sin.get_device() != device:
        raise ValueError(f"cos_sin must have shape (positions, rotary_dim), float32 or {q.dtype} on {q.device}, got "
                         f"{tuple(cos_sin.shape)}, {cos_sin.dtype} on {cos_sin.device}")
    table = cos_sin.data_ptr()
    if (table & 15 or not cos_sin.is_contiguous() or cos_sin.shape[1] & 7) and not _on16(cos_sin):
        raise ValueError("cos_sin must have a contiguous last axis and rows that start on 16 bytes")
    q, q_at, q_token, q_head = _placed_rows(q)
    k, k_at, k_token, k_head = _placed_rows(k)
    v, v_at, v_token, v_head = _placed_rows(v)
    if out is None:
        o = _new(q)
        o_token, o_head = shape[1] * dim, dim
    else:
        o = _out(out, shape, q)
        if not _on16(o):
            raise ValueError("out must have rows that start on 16 bytes")
        o_token, o_head = _row_strides(o)
    angles, rotary_dim = cos_sin.shape
    cache = _lib.KV_CACHE_ARGS.pack(
        k_at, v_at, k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scale), _lib.ptr(v_scale), slots.data_ptr(), k_token,
        k_head, v_token, v_head, *_row_strides(k_cache), *_row_strides(v_cache), shape[0], kv_heads, dim, pages, page, code,
        quantized)
    rotary = _lib.ROTARY_ARGS.pack(
        q_at, o.data_ptr(), positions.data_ptr(), table, q_token, q_head, o_token, o_head,
        cos_sin.stride(0) if angles > 1 else 0, shape[1], rotary_dim, angles, 0 if cos_sin.dtype == torch.float32 else code,
        bool(interleaved))
    return q, o, cache, rotary, (k, v, k_cache, v_cache, k_scale, v_scale, slots, positions, cos_sin)


def _rotary_launch(q, o, cache, rotary, _held):
    _lib.enqueue(_lib.load().cta_rotary_cache_write, q, cache, rotary)
    return o


def rotary_table(
    positions: int,
    rotary_dim: int,
    *,
    base: float = 10000.0,
    dtype: torch.dtype = torch.float32,
    device: Union[str, torch.device] = "cuda",
) -> torch.Tensor:
    """cos_sin [positions, rotary_dim] for ``rotary_cache_write``: the cosines, then the sines, of
    position / base**(2 i / rotary_dim), from angles in 64 bits (a position of 10^5 has
    no digits left behind the point of a turn in fp32), rounded once."""
    if positions < 0 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"positions must not be negative and rotary_dim even, got {positions} and {rotary_dim}")
    half = rotary_dim // 2
    turn = float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * turn
    return torch.cat([angle.cos(), angle.sin()], dim=1).to(dtype)


def kv_cache_read(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    *,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    dtype: Optional[torch.dtype] = None,
):
    """The rows k, v [T, kv_heads, dim] that slots [T] hold, as `dtype` (bf16 / fp16; None:
    the cache's own type, bf16 for e4m3); zeros for a negative slot.  One launch."""
    if k_cache.get_device() < 0:
        _require_cuda(k_cache, "k_cache")
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype == torch.float8_e4m3fn else k_cache.dtype
    sizes = _cache_sizes(k_cache, v_cache, k_scale, v_scale, dtype, k_cache)
    slots = _slots(slots, None, k_cache)
    # both in one allocation
    both = torch.empty((2, slots.shape[0], sizes[2], sizes[3]), dtype=dtype, device=k_cache.device)
    k, v = both.unbind(0)
    _cache_call(_lib.load().cta_kv_cache_read, k, v, k_cache, v_cache, slots, k_scale, v_scale, sizes)
    return k, v


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_rows: int = 1,
    scale: Optional[float] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
    shared_prefix: int = 0,
) -> torch.Tensor:
    """Attention of each sequence's newest rows over its keys and values in a paged cache
    (16-bit, or e4m3 with scales), those of the rows themselves included.

    q [T, heads, dim]; cu_seqlens (int32, B + 1) gives the rows of each of the B
    sequences, None one row each (decode).  seq_lens [B] (int32) counts all keys
    of a sequence, block_table [B, width] (int32) lists its pages.  Row r of n_r
    sees keys j <= seq_len - n_r + r.  Scales may be positive normal numbers of any size.
    Chunks over an e4m3 cache may be computed from a copy of the codes in 16 bits, in a
    workspace of up to 2 GiB.  max_rows, the longest n_r as the host knows it, only chooses
    the kernel.  No device data is read on the host.
    Rows that see no key are zero; rows behind the last sequence are not
    written.  A NaN or infinity in the v of a cached token may also reach earlier
    rows of this call.  A page outside the cache or a length past the table counts as no
    keys and is reported by ``_lib.device_error()``.

    `window`: the row whose last key is j0 sees the keys j <= j0 with j > j0 - window, and
    the first `sinks` keys.  Pages that no row sees are not read, and their entries in
    the table may hold anything: an engine may have freed them.

    `shared_prefix`: the batch's sequences all begin with the same keys, and the rows of
    block_table, also of sequences that end earlier, name the same pages for the first
    shared_prefix of them (a page that they fill in part does not count).  Where that pays they are read once for all
    rows; it changes what the call costs, and its sums' order, not what it computes.
    It serves single tokens and a few per sequence; chunks of many rows, and calls with a window, are as without it.  A NaN or infinity in the v of a shared key may then also reach
    sequences that end before it."""
    return _paged_launch(*_paged_plan(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens, max_rows, scale, k_scale,
                                      v_scale, out, window, sinks, shared_prefix))


def _paged_plan(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens, max_rows, scale, k_scale, v_scale, out,
                window=None, sinks=0, shared_prefix=0):
    """All checks of paged_attention, and what its launch takes: (q, out, the library's call, its arguments, bytes of
    workspace, the tensors that the arguments point to)."""
    reach = _window(window, sinks)
    prefix = operator.index(shared_prefix)
    if prefix < 0:
        raise ValueError(f"shared_prefix must not be negative, got {prefix}")
    device = q.get_device()
    if device < 0:
        _require_cuda(q, "q")
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("q must have shape (T, heads, dim)")
    code = _lib.dtype_code(q.dtype)
    pages, page, kv_heads, dim, quantized = _cache_sizes(k_cache, v_cache, k_scale, v_scale, q.dtype, q)
    rows, heads, q_dim = shape
    if q_dim != dim or heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not go with a cache {tuple(k_cache.shape)}")
    table, lens = block_table, seq_lens
    if table.dtype != torch.int32 or table.get_device() != device:
        table = _device_ints(table, "block_table", q, torch.int32)
    if lens.dtype != torch.int32 or lens.get_device() != device:
        lens = _device_ints(lens, "seq_lens", q, torch.int32)
    tshape, lshape = table.shape, lens.shape
    if len(tshape) != 2 or len(lshape) != 1 or tshape[0] != lshape[0]:
        raise ValueError("block_table must have shape (B, width), seq_lens (B,)")
    if table.stride(1) != 1:
        table = table.contiguous()
    if not lens.is_contiguous():
        lens = lens.contiguous()
    batch = lshape[0]
    cu = None
    if cu_seqlens is not None:
        cu = _offsets(cu_seqlens, q)
        if cu.shape[0] != batch + 1:
            raise ValueError(f"cu_seqlens must have {batch + 1} entries, got {cu.shape[0]}")
    q, q_at, q_token, q_head = _placed_rows(q)
    if out is None:
        o = _new(q)
        o_token, o_head = heads * dim, dim
    else:
        o = _out(out, shape, q)
        if not _on16(o):
            raise ValueError("out must have rows that start on 16 bytes")
        o_token, o_head = _row_strides(o)
    lib = _lib.load()
    args = _lib.PAGED_ATTENTION_ARGS.pack(
        q_at, o.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scale), _lib.ptr(v_scale),
        table.data_ptr(), lens.data_ptr(), _lib.ptr(cu), q_token, q_head, o_token, o_head, *_row_strides(k_cache),
        *_row_strides(v_cache), table.stride(0), rows, batch, heads, kv_heads, dim, pages, page, tshape[1],
        int(max_rows), code, quantized, dim**-0.5 if scale is None else float(scale), 0.0)
    if reach[0]:
        fn, query, args = lib.cta_window_paged_attention, lib.cta_window_paged_attention_workspace_bytes, (args, *reach)
    elif prefix:
        fn, query, args = lib.cta_prefix_paged_attention, lib.cta_prefix_paged_attention_workspace_bytes, (args, prefix)
    else:
        fn, query, args = lib.cta_paged_attention, lib.cta_paged_attention_workspace_bytes, (args,)
    nbytes = _workspace_bytes(query, q, *args)
    return q, o, fn, args, nbytes, (k_cache, v_cache, k_scale, v_scale, table, lens, cu)


def _paged_launch(q, o, fn, args, nbytes, _held):
    # a buffer of the caching allocator per call: calls on other streams and captured graphs have their own
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _lib.enqueue(fn, q, *args, _lib.ptr(ws), nbytes)
    return o
