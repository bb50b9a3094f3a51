"""8-bit activation checkpoints, and the linear layer that keeps its input as one.

What training holds between forward and backward is mostly activations.  A checkpoint holds one of
them in a byte an element: 32 consecutive channels of a row share a power-of-two scale 2^e, the
smallest with ``max|x| <= 127 * 2^e``, and an element is ``round(x / 2^e)`` (to nearest, ties to
even), so a value is off by at most ``max|x| / 127`` of its block.  (What the last half step of a type's
range rounds up to, the type does not hold: it comes back as the largest finite value.)  A block that holds an infinity or
a NaN comes back as NaN.  Kernels: ``csrc/kernels/ckpt8.hip``, ``csrc/kernels/linear_ckpt8_*.hip``
(format: ``csrc/include/rtseg_ckpt8.h``).

* :func:`ckpt8_pack` / :func:`ckpt8_unpack`: a tensor to its checkpoint and back.
* :func:`ckpt8_saved`: a context in which operators that save a tensor for their backward save its
  checkpoint instead (the Mix-FFN's depth-wise conv, the attention's spatial-reduction conv).
* :func:`linear_ckpt8`: ``act(x) @ weight.T + bias``.  The forward is that of the exact ``x``; it
  writes the checkpoint while it stages ``x``, and both gradients read the checkpoint on the fly: the
  weight gradient's MFMA operands are decoded in front of LDS, the activation is recomputed from the
  codes, so neither ``x`` nor ``act(x)`` is held.
* :func:`convert_ckpt8`: a model's linear layers, layer norms and Mix Transformer convs onto 8-bit
  checkpoints (``config.act_ckpt8``).

Reference: the Mix Transformer encoders of the reference's segmentation_models_pytorch bridge
(reference models/__init__.py:67-81), whose blocks are such layers.  CPU tensors and
``RTSEG_DISABLE_HIP=1`` / ``RTSEG_HIP_OFF=ckpt8`` run the same formulas, checkpoint included, in PyTorch.
"""
from __future__ import annotations

import contextlib
import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ._ext import differentiable_once, ops, transformed, use_hip

BLOCK = 32
ACTS = {"none": 0, "gelu": 1}
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class Ckpt8(NamedTuple):
    """``codes`` int8 ``[rows, padded channels]``, ``scales`` uint8 ``[rows, padded channels / 32]`` (the
    exponent + 127), and the shape and type of the tensor that they stand for."""

    codes: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]
    shape: torch.Size
    dtype: torch.dtype


def _pack_reference(x2: torch.Tensor):
    rows, c = x2.shape
    cp = c + -c % BLOCK
    v = F.pad(x2.float(), (0, cp - c)).view(rows, cp // BLOCK, BLOCK)
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    mant, expo = torch.frexp(torch.where(bad, torch.zeros_like(amax), amax))
    e = (expo - 7 + (mant > 127 / 128)).clamp_min(-126)
    e = torch.where(mant == 0, torch.full_like(e, -126), e)
    q = torch.ldexp(v, -e.unsqueeze(-1)).round()
    q = torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127)
    return q.to(torch.int8).view(rows, cp), scales.to(torch.uint8)


def _unpack_reference(codes, scales, c, dtype, held=torch.float32):
    """``held``: the type of the tensor that was packed."""
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.to(torch.int32) - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    v = codes.float().view(*scales.shape, BLOCK) * s.unsqueeze(-1)
    v = v.clamp(torch.finfo(held).min, torch.finfo(held).max)  # NaN stays NaN
    return v.view(codes.shape)[:, :c].to(dtype)


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: the last axis must have at least one channel, got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: fp32, bf16 or fp16 expected, got {x.dtype}")
    return x.reshape(-1, x.shape[-1]).contiguous()


def ckpt8_pack(x: torch.Tensor) -> Ckpt8:
    """The 8-bit checkpoint of ``x`` (``[..., C]``, fp32 / bf16 / fp16), blocked along the last axis.
    Not differentiable: it holds values, as ``save_for_backward`` does."""
    x2 = _rows(x.detach(), "ckpt8_pack")
    codes, scales = ops().ckpt8_pack(x2) if use_hip(x2, "ckpt8") else _pack_reference(x2)
    return Ckpt8(codes, scales, x.shape, x.dtype)


def ckpt8_unpack(ckpt: Ckpt8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The tensor that ``ckpt`` stands for, in its own type or ``dtype``."""
    dtype = dtype or ckpt.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"ckpt8_unpack: fp32, bf16 or fp16 expected, got {dtype}")
    c = ckpt.shape[-1]
    f = ops().ckpt8_unpack if use_hip(ckpt.codes, "ckpt8") else _unpack_reference
    return f(ckpt.codes, ckpt.scales, c, dtype, ckpt.dtype).view(ckpt.shape)


@contextlib.contextmanager
def ckpt8_saved(x: Optional[torch.Tensor]):
    """Inside, whatever an operator saves of ``x`` for its backward -- ``x`` or a view of all of it -- is
    held as an 8-bit checkpoint and decoded when the backward asks for it; every other saved tensor
    stays as it is.  4-D channels-last tensors are blocked along their channels, others along the last
    axis.  ``None``, a tensor of another type, one that carries no gradient, or a call that is traced or
    transformed: nothing changes."""
    if (x is None or x.dtype not in _DTYPES or not (torch.is_grad_enabled() and x.requires_grad and x.numel())
            or transformed(x)):
        yield
        return

    # the hooks live as long as what they packed: they know x by these values, not by a reference that
    # would hold it (x itself lives at least as long as this context)
    who = (x.dtype, x.numel(), x.data_ptr(), x.device)

    def pack(t):
        if (t.dtype, t.numel(), t.data_ptr(), t.device) != who or isinstance(t, nn.Parameter):
            return t, t._version  # autograd leaves the check for changes in place to the hooks
        last = t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last) and not t.is_contiguous()
        return last, ckpt8_pack(t.permute(0, 2, 3, 1) if last else t)

    def unpack(held):
        if isinstance(held[0], torch.Tensor):
            t, version = held
            if t._version != version:
                raise RuntimeError(
                    "ckpt8_saved: one of the variables needed for gradient computation has been modified by an inplace "
                    f"operation: a tensor of shape {tuple(t.shape)} is at version {t._version}, expected version {version}")
            return t
        last, ckpt = held
        v = ckpt8_unpack(ckpt)
        return v.permute(0, 3, 1, 2) if last else v

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        yield


# ---------------------------------------------------------------------------------- linear


def _gelu(v):
    """The erf form in an order that holds at the largest values (2 v is not formed)."""
    return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))


def _gelu_slope(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def linear_ckpt8_reference(x2, weight, bias, act):
    """Forward of :func:`linear_ckpt8` in PyTorch: the activation rounded to ``x``'s type, the product
    and its operands in that type."""
    a = _gelu(x2.float()).to(x2.dtype) if act == "gelu" else x2
    with torch.autocast(x2.device.type, enabled=False):
        return F.linear(a, weight.to(x2.dtype), None if bias is None else bias.to(x2.dtype))


class _LinearCkpt8Fn(torch.autograd.Function):
    """The PyTorch formulation (CPU tensors)."""

    @staticmethod
    def forward(ctx, x2, weight, bias, act):
        need_x, need_w = ctx.needs_input_grad[:2]
        keep = need_w or (need_x and act != "none")
        codes, scales = _pack_reference(x2) if keep else (None, None)
        ctx.act, ctx.k, ctx.wtype = act, x2.shape[1], weight.dtype
        ctx.save_for_backward(codes, scales, weight if need_x else None)
        return linear_ckpt8_reference(x2, weight, bias, act)

    @staticmethod
    @differentiable_once
    def backward(ctx, dy):
        codes, scales, weight = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = dw = db = None
        z = None if codes is None else _unpack_reference(codes, scales, ctx.k, torch.float32, dy.dtype)
        g = dy.float()
        with torch.autocast(dy.device.type, enabled=False):  # the backward may be called inside of one
            if need_x:
                dx = g @ weight.to(dy.dtype).float()
                dx = (dx * _gelu_slope(z) if ctx.act == "gelu" else dx).to(dy.dtype)
            if need_w:
                a = _gelu(z).to(dy.dtype).float() if ctx.act == "gelu" else z
                dw = (g.t() @ a).to(ctx.wtype)
            if need_b:
                db = g.sum(0).to(ctx.wtype)
        return dx, dw, db, None


def linear_ckpt8(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 act: str = "none") -> torch.Tensor:
    """``act(x) @ weight.T + bias`` that keeps ``x`` for the backward as an 8-bit checkpoint.

    ``x``: ``[..., in]`` fp32 / bf16 / fp16; under autocast it is cast to the autocast type, as
    ``F.linear`` would.  ``weight`` ``[out, in]`` and ``bias`` ``[out]`` are of ``x``'s type or fp32 (master
    weights: the products are taken in ``x``'s type, the gradients come in fp32).  ``act``: ``"none"`` or
    ``"gelu"`` (the erf form, applied in fp32 and rounded to ``x``'s type, as a layer of its own would).
    The value is that of the exact ``x``; the gradients are the formula's at the checkpoint's values:
    ``dx = (dy @ weight) * act'(z)``, ``dweight = dy.T @ act(z)``, ``dbias = dy.sum(rows)``.
    Without gradients nothing is kept.  A call that is traced, compiled or transformed (``torch.func``, forward
    mode) takes the formula itself, without a checkpoint."""
    if act not in ACTS:
        raise ValueError(f"linear_ckpt8: act must be one of {sorted(ACTS)}, got {act!r}")
    if weight.dim() != 2 or min(weight.shape) < 1 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_ckpt8: weight must be [out, in] for x [..., in], got {tuple(weight.shape)} "
                         f"for {tuple(x.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"linear_ckpt8: bias must have shape ({weight.shape[0]},), got {tuple(bias.shape)}")
    kind = x.device.type
    if torch.is_autocast_enabled(kind) and x.dtype in _DTYPES:  # autocast leaves fp64 alone
        x = x.to(torch.get_autocast_dtype(kind))
    if x.dtype not in _DTYPES:
        raise TypeError(f"linear_ckpt8: fp32, bf16 or fp16 expected, got {x.dtype}")
    if bias is not None and bias.dtype != weight.dtype:
        raise TypeError(f"linear_ckpt8: weight and bias must be of one type, got {weight.dtype} and {bias.dtype}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"linear_ckpt8: weight must be of x's type ({x.dtype}) or fp32, got {weight.dtype}")
    for p in (weight, bias):
        if p is not None and p.device != x.device:
            raise ValueError(f"linear_ckpt8: all tensors must be on one device, got {x.device} and {p.device}")
    if transformed(x):  # traced, compiled, torch.func, forward mode: the formulation itself, without a checkpoint
        y = linear_ckpt8_reference(_rows(x, "linear_ckpt8"), weight, bias, act)
        return y.view(*x.shape[:-1], weight.shape[0])
    if use_hip(x, "ckpt8"):
        return ops().linear_ckpt8(x, weight, bias, ACTS[act])
    y = _LinearCkpt8Fn.apply(_rows(x, "linear_ckpt8"), weight, bias, act)
    return y.view(*x.shape[:-1], weight.shape[0])


class Ckpt8Linear(nn.Linear):
    """``nn.Linear`` on :func:`linear_ckpt8`; parameters and state_dict keys unchanged.
    ``forward(x, act="gelu")`` is ``self(gelu(x))`` in one layer."""

    def forward(self, x, act="none"):
        return linear_ckpt8(x, self.weight, self.bias, act)


def convert_ckpt8(model: nn.Module) -> nn.Module:
    """Hold the activations of ``model``'s linear layers, layer norms and Mix Transformer convs in 8
    bits (in place; classes and flags only -- parameters and checkpoint keys are unchanged)."""
    from .layer_norm import convert_layernorm

    convert_layernorm(model)
    for m in model.modules():
        if type(m) is nn.Linear:
            m.__class__ = Ckpt8Linear
        elif hasattr(type(m), "ckpt8"):
            m.ckpt8 = True
    return model


__all__ = ["Ckpt8", "ckpt8_pack", "ckpt8_unpack", "ckpt8_saved", "linear_ckpt8", "linear_ckpt8_reference", "Ckpt8Linear", "convert_ckpt8"]
