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


def rms_norm(x, weight, *, residual=None, eps: float = 1e-6, out_dtype=None):
    """``y = t * rsqrt(mean(t^2) + eps) * weight`` over the last axis with ``t = x`` or ``x + residual``.

    ``x`` and ``residual`` ``[..., dim]`` in one of bf16, f16 and f32, ``weight [dim]``; ``dim`` up to 16384. Returns ``y`` in
    ``x``'s dtype, with a residual ``(y, stream)`` where ``stream = t`` rounded to that dtype (``y`` is taken of the unrounded
    sum). ``out_dtype=torch.float8_e4m3fn`` returns ``(q, scale)`` or ``(q, scale, stream)`` instead: ``scale [...]`` float32 is
    the row's largest ``|y|`` over 448 (1 for a row of zeros), ``q * scale`` stands for ``y``. That form has no gradient and is
    refused where one would be recorded.
    """
    out = (_lib._torch_ops or _lib.torch_ops()).rms_norm(x, weight, residual, eps, out_dtype)
    if out is not None:
        return out
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("rms_norm runs on CUDA tensors only: the 'cuda' implementation has no CPU fallback")
    if x.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {x.dtype}")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= 16384:
        raise ValueError(f"x must be [..., dim] with 1 <= dim <= 16384; got {tuple(x.shape)}")
    if not isinstance(weight, torch.Tensor) or weight.shape != x.shape[-1:] or weight.device != x.device or not weight.is_floating_point():
        raise ValueError(f"weight must be a floating [{x.shape[-1]}] on {x.device}; got "
                         f"{weight if not isinstance(weight, torch.Tensor) else (weight.dtype, tuple(weight.shape), weight.device)}")
    if residual is not None and not isinstance(residual, torch.Tensor):
        raise ValueError(f"residual must be a tensor or None; got {type(residual).__name__}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual must be {x.dtype} {tuple(x.shape)} on {x.device}; got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    if out_dtype not in (None, x.dtype, torch.float8_e4m3fn):
        raise ValueError(f"out_dtype must be {x.dtype} or torch.float8_e4m3fn; got {out_dtype}")
    raise ValueError("an e4m3 output has no gradient: call rms_norm under torch.no_grad(), or with out_dtype=None")
