"""The norms of a block: ``gated_rms_norm`` behind the linear-attention kernels and ``rms_norm`` of the residual stream in
front of a mixer or a feed-forward block.

``rms_norm`` (the reference's plain norm is ``RMSNorm`` in ``src/jla/layers/norm.py``) adds the residual before it takes the
norm, ``t = x + residual``, and hands the sum back as the new residual stream; it can leave its output in e4m3 with one
scale a row for ``linear`` and ``gated_linear``. One pass over the rows forward and one backward (``jla_rms_norm_fwd/bwd``).

Gated RMS norm after the linear-attention kernels (mirror of ``GatedRMSNorm`` in the reference's
``src/jla/layers/norm.py:60-112``), one fused CUDA pass forward and one backward (``jla_gated_rmsnorm_fwd/bwd``).

``norm_before_gate=True``: ``rms_norm(x) * weight * act(z)`` (Gated DeltaNet with ``activation="silu"``, KDA with
``"sigmoid"``); ``False``: ``rms_norm(x * act(z)) * weight`` (Mamba-2). ``group_size`` normalises each group of that
many consecutive channels of the last axis on its own (``None``: the whole axis). Computed in float32, returned in
``x``'s dtype.
"""

from __future__ import annotations

import ctypes as C

import torch

from .. import _lib
from ..ops.cuda import aligned, nothing_to_differentiate

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _call(name, x, *args):
    _lib.launch(name, x.device, *args)


def _ptr(t):
    return t.data_ptr()


class _GatedRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, weight, eps, sigmoid_gate, norm_before_gate, group):
        dim = x.shape[-1]
        rows = x.numel() // dim
        y = torch.empty_like(x)
        _call("jla_gated_rmsnorm_fwd", x, _DTYPES[x.dtype], rows, dim, group, _ptr(x), _ptr(z), _ptr(weight),
              eps, int(sigmoid_gate), int(norm_before_gate), _ptr(y))
        ctx.save_for_backward(x, z, weight)
        ctx.cfg = (eps, sigmoid_gate, norm_before_gate, group)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, z, weight = ctx.saved_tensors
        eps, sigmoid_gate, norm_before_gate, group = ctx.cfg
        dim = x.shape[-1]
        rows = x.numel() // dim
        dy = dy.contiguous()
        dx, dz, dw = torch.empty_like(x), torch.empty_like(z), torch.empty_like(weight)
        _call("jla_gated_rmsnorm_bwd", x, _DTYPES[x.dtype], rows, dim, group, _ptr(x), _ptr(z), _ptr(weight),
              eps, int(sigmoid_gate), int(norm_before_gate), _ptr(dy), _ptr(dx), _ptr(dz), _ptr(dw))
        return dx, dz, dw, None, None, None, None


def gated_rms_norm(x, z, weight, *, eps: float = 1e-6, activation: str = "silu", norm_before_gate: bool = True,
                   group_size: int | None = None):
    """``GatedRMSNorm(dim, eps=..., activation=..., norm_before_gate=..., group_size=...)(x, z)`` with ``weight [dim]``."""
    if activation not in ("silu", "sigmoid"):
        raise ValueError(f"unsupported gate activation {activation!r}")
    if z.shape != x.shape:
        raise ValueError(f"gate shape {tuple(z.shape)} must match input shape {tuple(x.shape)}")
    dim = x.shape[-1]
    group = group_size or dim
    if group < 1 or dim % group:
        raise ValueError(f"group_size {group_size} must divide dim {dim}")
    if weight.shape != (dim,):
        raise ValueError(f"weight must be [{dim}]; got {tuple(weight.shape)}")
    if not x.is_cuda:
        raise ValueError("gated_rms_norm runs on CUDA tensors only: the 'cuda' implementation has no CPU fallback")
    if x.dtype not in _DTYPES or z.dtype != x.dtype:
        raise ValueError(f"x and z must share one of {sorted(str(d) for d in _DTYPES)}; got {x.dtype}, {z.dtype}")
    return _GatedRMSNorm.apply(x.contiguous(), z.contiguous(), weight.float().contiguous(), float(eps),
                               activation == "sigmoid", bool(norm_before_gate), int(group))


class _RMSNorm(torch.autograd.Function):
    """``(y, stream)``; ``stream`` is None without a residual."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, stream, rstd, _ = _rms_norm_fwd(x, residual, weight, eps, False, True)
        ctx.save_for_backward(x, residual, rstd, weight)
        ctx.set_materialize_grads(False)
        if stream is not None and not (ctx.needs_input_grad[0] or ctx.needs_input_grad[1]):
            ctx.mark_non_differentiable(stream)  # the weight is not in it
        return y, stream

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstream):
        x, residual, rstd, weight = ctx.saved_tensors
        if dy is None:  # only the stream was used
            return dstream, dstream, None, None
        dim = x.shape[-1]
        rows = x.numel() // dim
        dy, dstream = aligned(dy), aligned(dstream)
        dx = torch.empty_like(x)
        dw = scratch = None
        if ctx.needs_input_grad[2]:
            dw = torch.empty_like(weight)
            nbytes = _lib.load().jla_rms_norm_bwd_scratch_bytes(rows, dim)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        _lib.launch("jla_rms_norm_bwd", x.device, _DTYPES[x.dtype], rows, dim, _ptr(x),
                    None if residual is None else _ptr(residual), _ptr(rstd), _ptr(weight), _ptr(dy),
                    None if dstream is None else _ptr(dstream), _ptr(dx), None if dw is None else _ptr(dw),
                    None if scratch is None else _ptr(scratch), 0 if scratch is None else scratch.numel())
        return dx, dx if ctx.needs_input_grad[1] else None, dw, None


def _rms_norm_fwd(x, residual, weight, eps, e4m3, keep_rstd):
    dim, device = x.shape[-1], x.device
    rows = x.numel() // dim
    y = torch.empty_like(x, dtype=torch.float8_e4m3fn) if e4m3 else torch.empty_like(x)
    stream = None if residual is None else torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=device) if keep_rstd else None
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=device) if e4m3 else None
    _lib.launch("jla_rms_norm_fwd", device, _DTYPES[x.dtype], rows, dim, x.data_ptr(),
                None if residual is None else residual.data_ptr(), weight.data_ptr(), eps, e4m3, y.data_ptr(),
                None if stream is None else stream.data_ptr(), None if rstd is None else rstd.data_ptr(),
                None if scale is None else scale.data_ptr())
    return y, stream, rstd, scale


def rms_norm(x, weight, *, residual=None, eps: float = 1e-6, out_dtype=None):
    """``y = t * rsqrt(mean(t^2) + eps) * weight`` over the last axis with ``t = x`` or ``x + residual``.

    ``x`` and ``residual`` ``[..., dim]`` in one of bf16, f16 and f32, ``weight [dim]``; ``dim`` up to 16384. Returns ``y`` in
    ``x``'s dtype, with a residual ``(y, stream)`` where ``stream = t`` rounded to that dtype (``y`` is taken of the unrounded
    sum). ``out_dtype=torch.float8_e4m3fn`` returns ``(q, scale)`` or ``(q, scale, stream)`` instead: ``scale [...]`` float32 is
    the row's largest ``|y|`` over 448 (1 for a row of zeros), ``q * scale`` stands for ``y``. That form has no gradient and is
    refused where one would be recorded.
    """
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("rms_norm runs on CUDA tensors only: the 'cuda' implementation has no CPU fallback")
    if x.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= 16384:
        raise ValueError(f"x must be [..., dim] with 1 <= dim <= 16384; got {tuple(x.shape)}")
    if weight.shape != x.shape[-1:] or weight.device != x.device:
        raise ValueError(f"weight must be [{x.shape[-1]}] on {x.device}; got {tuple(weight.shape)} on {weight.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual must be {x.dtype} {tuple(x.shape)} on {x.device}; got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    e4m3 = out_dtype == torch.float8_e4m3fn
    if out_dtype is not None and not e4m3 and out_dtype != x.dtype:
        raise ValueError(f"out_dtype must be {x.dtype} or torch.float8_e4m3fn; got {out_dtype}")
    plain = nothing_to_differentiate((x, weight, residual))
    if e4m3 and not plain:
        raise ValueError("an e4m3 output has no gradient: call rms_norm under torch.no_grad(), or with out_dtype=None")
    x, weight, residual = aligned(x), aligned(weight if weight.dtype is torch.float32 else weight.float()), aligned(residual)
    if plain:
        y, stream, _, scale = _rms_norm_fwd(x, residual, weight, float(eps), e4m3, False)
    else:
        (y, stream), scale = _RMSNorm.apply(x, residual, weight, float(eps)), None
    out = (y,) if scale is None else (y, scale)
    out = out if stream is None else (*out, stream)
    return out[0] if len(out) == 1 else out
