"""Layer norm over the last axis on the HIP kernels of ``csrc/kernels/layer_norm_*.hip``.

Reference: the Mix Transformer encoders that the reference reaches through
segmentation_models_pytorch (reference models/__init__.py:67-81) normalise every token of the
residual stream twice per block (``nn.LayerNorm``).  Here the sum of the residual stream and a
branch, the norm and the cast to the next linear layer's type are one pass, and the backward is one
pass that also adds the stream's own gradient and reduces the weight gradients (fp32, without
atomics: the same bits on every run).

``ckpt8=True`` holds the normalised tensor for the backward as an 8-bit checkpoint (``ops.ckpt8``)
instead of the tensor itself.  CPU tensors, ``RTSEG_DISABLE_HIP=1`` / ``RTSEG_HIP_OFF=layer_norm``
and more than 8192 channels run the same formulas in PyTorch; so does a call that is traced, compiled or
transformed (``torch.func``, forward mode), without a checkpoint.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ._ext import differentiable_once, ops, transformed, use_hip

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_MAX_CHANNELS = 8192  # a row is held in one block's registers


def _autocast_dtype(t: torch.Tensor) -> Optional[torch.dtype]:
    kind = t.device.type
    return torch.get_autocast_dtype(kind) if torch.is_autocast_enabled(kind) else None


def _default_out(x: torch.Tensor) -> torch.dtype:
    """What ``F.layer_norm`` returns: fp32 under autocast, which leaves fp64 alone, else the input's type."""
    return torch.float32 if x.dtype != torch.float64 and _autocast_dtype(x) is not None else x.dtype


def layer_norm_reference(x, weight=None, bias=None, eps=1e-5, residual=None, out_dtype=None):
    """The formulas of :func:`layer_norm` in PyTorch (statistics in fp32, or in fp64 for fp64 inputs)."""
    out_dtype = out_dtype or x.dtype
    s = x if residual is None else x + residual
    wide = s.dtype if s.dtype == torch.float64 else torch.float32
    with torch.autocast(s.device.type, enabled=False):
        y = F.layer_norm(s.to(wide), s.shape[-1:], None if weight is None else weight.to(wide),
                         None if bias is None else bias.to(wide), eps).to(out_dtype)
    return y if residual is None else (s, y)


class _LayerNormCkptFn(torch.autograd.Function):
    """The PyTorch formulation with an 8-bit checkpoint (CPU tensors)."""

    @staticmethod
    def forward(ctx, s, weight, bias, eps, out_dtype):
        from .ckpt8 import ckpt8_pack

        wide = s.detach().float()
        mean = wide.mean(-1, keepdim=True)
        mean = mean + (wide - mean).mean(-1, keepdim=True)  # what the sum's roundings left out, as in the kernel
        rstd = torch.rsqrt((wide - mean).square().mean(-1, keepdim=True) + eps)
        h = (wide - mean) * rstd
        if weight is not None:
            h = h * weight.float()
        if bias is not None:
            h = h + bias.float()
        kept = ckpt8_pack(s.detach())
        ctx.kept = kept._replace(codes=None, scales=None)
        ctx.save_for_backward(kept.codes, kept.scales, mean, rstd, weight)
        ctx.bias_type = None if bias is None else bias.dtype
        return h.to(out_dtype)

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        from .ckpt8 import ckpt8_unpack

        codes, scales, mean, rstd, weight = ctx.saved_tensors
        x = ckpt8_unpack(ctx.kept._replace(codes=codes, scales=scales))
        h = (x.float() - mean) * rstd
        dy = dy.float()
        g = dy if weight is None else dy * weight.float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
        lead = tuple(range(dy.dim() - 1))
        return (dx.to(x.dtype) if ctx.needs_input_grad[0] else None,
                (dy * h).sum(lead).to(weight.dtype) if ctx.needs_input_grad[1] else None,
                dy.sum(lead).to(ctx.bias_type) if ctx.needs_input_grad[2] else None, None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
               ckpt8: bool = False, want_sum: bool = True):
    """``y = (s - mean) * rsqrt(var + eps) * weight + bias`` over the last axis, ``s = x``; with
    ``residual`` the pair ``(s, y)`` for ``s = x + residual`` (``want_sum=False``: ``(None, y)``).

    ``x``: ``[..., C]`` fp32 / bf16 / fp16, any strides (a non-contiguous one is copied once).  ``s``
    has the promoted type of ``x`` and ``residual``; ``y`` has ``out_dtype``, by default fp32 under
    autocast (fp64 stays fp64) and the type of ``s`` otherwise (as ``F.layer_norm`` on the GPU).  ``weight`` / ``bias``: ``[C]`` or
    None, applied in fp32.  ``ckpt8``: hold ``s`` for the backward in 8 bits; the backward then uses
    the checkpoint's values in place of ``s`` (with the exact mean and variance).
    """
    c = x.shape[-1] if x.dim() else 0
    if c < 1:
        raise ValueError(f"layer_norm: the last axis must have at least one channel, got shape {tuple(x.shape)}")
    if not x.is_floating_point():
        raise TypeError(f"layer_norm: x must be of a floating type, got {x.dtype}")
    if residual is not None and not residual.is_floating_point():
        raise TypeError(f"layer_norm: residual must be of a floating type, got {residual.dtype}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and tuple(p.shape) != (c,):
            raise ValueError(f"layer_norm: {name} must have shape ({c},), got {tuple(p.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"layer_norm: residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if out_dtype is not None and not out_dtype.is_floating_point:
        raise ValueError(f"layer_norm: out_dtype must be a floating type, got {out_dtype}")
    if residual is not None:
        wide = torch.promote_types(x.dtype, residual.dtype)
        if x.dtype != wide:
            x = x.to(wide)
        # an fp32 stream takes a 16-bit branch as it is; every other pair is added in one type
        if residual.dtype != wide and not (wide == torch.float32 and residual.dtype in _DTYPES):
            residual = residual.to(wide)
    out_dtype = out_dtype or _default_out(x)
    stock = transformed(x)
    if not stock and x.dtype in _DTYPES and out_dtype in _DTYPES and c <= _MAX_CHANNELS and use_hip(x, "layer_norm"):
        # 16 bits in and another 16-bit type out: through fp32
        got = out_dtype if out_dtype == x.dtype or torch.float32 in (out_dtype, x.dtype) else torch.float32
        *s, y = ops().layer_norm(x, residual, weight, bias, eps, got, ckpt8, residual is not None and want_sum)
        y = y if got == out_dtype else y.to(out_dtype)
        return y if residual is None else (s[0] if s else None, y)
    if ckpt8 and not stock and x.dtype in _DTYPES and torch.is_grad_enabled():
        s = x if residual is None else x + residual
        y = _LayerNormCkptFn.apply(s, weight, bias, float(eps), out_dtype)
        return y if residual is None else (s if want_sum else None, y)
    got = layer_norm_reference(x, weight, bias, eps, residual, out_dtype)
    return got if residual is None or want_sum else (None, got[1])


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one axis on :func:`layer_norm`; parameters and state_dict keys unchanged.

    ``forward(x)`` is the stock module's.  ``forward(x, residual=r)`` returns ``(x + r, norm(x + r))``,
    ``out_dtype`` sets the result's type, and ``ckpt8`` (an attribute, off) holds the normalised tensor
    in 8 bits for the backward."""

    ckpt8 = False

    def forward(self, x, residual=None, out_dtype=None, want_sum=True):
        if len(self.normalized_shape) != 1:
            if residual is not None or out_dtype is not None:
                raise ValueError("LayerNorm: residual / out_dtype need a norm over the last axis alone")
            return super().forward(x)
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm: {self.normalized_shape[0]} channels expected, got shape {tuple(x.shape)}")
        if x.device.type != "cuda" and residual is None and out_dtype is None and not self.ckpt8:
            return super().forward(x)
        return layer_norm(x, self.weight, self.bias, self.eps, residual, out_dtype, self.ckpt8, want_sum)


def convert_layernorm(model: nn.Module) -> nn.Module:
    """Swap every ``nn.LayerNorm`` of ``model`` onto :class:`LayerNorm` (in place)."""
    for m in model.modules():
        if type(m) is nn.LayerNorm:
            m.__class__ = LayerNorm
    return model


__all__ = ["layer_norm", "layer_norm_reference", "LayerNorm", "convert_layernorm"]
