"""64-bit references of the token operators (layer norm, 8-bit checkpoints, checkpointing linear layer) and
the error bounds that a correct kernel keeps.

u = 2^-24 is half a step of fp32 relative to the value, EPS[t] = finfo(t).eps / 2 that of the output type:
a result is off by its own rounding (EPS * |value|) plus what fp32 sums cost.  A sum of n fp32 terms in any
order is off by at most n * u * sum |terms|.
"""
import math

import torch

U = 2.0 ** -24
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}  # half a subnormal step


def check(got, ref, tol, what=""):
    """|got - ref| <= tol element by element; NaN where ref has NaN, infinities as ref has them."""
    got, ref, tol = got.detach().double().cpu(), ref.detach().double().cpu(), tol.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)]), what
    d = (got - ref).abs()[fin]
    t = tol.expand_as(ref)[fin]
    bad = d > t
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / t).max()):.3g} x the bound"


def checkpoint(x):
    """What the 8-bit checkpoint of x [rows, c] stands for, in fp64 (finite x)."""
    rows, c = x.shape
    cp = c + -c % 32
    b = torch.nn.functional.pad(x.double(), (0, cp - c)).view(rows, cp // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)) / 127)).clamp_min(-126)
    e = torch.where(amax > 0, e, torch.full_like(e, -126))
    return (torch.round(b * torch.exp2(-e)) * torch.exp2(e)).view(rows, cp)[:, :c]


def gelu(v):
    return v * torch.special.ndtr(v)


def gelu_slope(v):
    return torch.special.ndtr(v) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)


class NormRef:
    """s, y and the gradients of layer_norm in fp64, with their bounds.

    A row's statistics are sums of c terms, added up as at most 32 in a lane and 8 levels of a tree: 41 u
    with the division.  mean: 41 u A for A = max |s|.  h = (s - mean) * rstd: the mean's error and one
    rounding of the difference, (42 u A) * rstd, and rstd's relative error -- the variance's 45 u, halved,
    plus the mean's second-order part and 3 roundings -- 30 u on |h| <= 2 A rstd: below 102 u A rstd =: EH."""

    def __init__(self, x, w, b, eps, residual=None, out=None, dy=None, ds=None, ckpt=False):
        out = out or x.dtype
        wide = x.dtype if residual is None else torch.promote_types(x.dtype, residual.dtype)
        s = x.detach().double() if residual is None else (x.detach().double() + residual.detach().double()).to(wide).double()
        c = s.shape[1]
        self.s = s
        mean = s.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((s - mean).square().mean(1, keepdim=True) + eps)
        wd = torch.ones(c, dtype=torch.float64, device=s.device) if w is None else w.detach().double()
        bd = torch.zeros(c, dtype=torch.float64, device=s.device) if b is None else b.detach().double()
        h = (s - mean) * rstd
        self.y = h * wd + bd
        A = s.abs().amax(1, keepdim=True)
        eh = 102 * U * A * rstd
        self.y_tol = EPS[out] * self.y.abs() + eh * wd.abs() + 3 * U * (self.y.abs() + bd.abs()) + TINY[out]
        if dy is None:
            return
        dy = dy.double()
        if ckpt:
            z = checkpoint(s)
            h = (z - mean) * rstd
            eh = 102 * U * torch.maximum(A, z.abs().amax(1, keepdim=True)) * rstd
        g = dy * wd
        c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
        dx = rstd * (g - c1 - h * c2)
        G, H = g.abs().amax(1, keepdim=True), h.abs().amax(1, keepdim=True)
        # c1: 43 u G; c2: 43 u G H + G EH; h c2: EH |c2| + H * (c2's error); 3 roundings and rstd's 30 u on each term
        e = rstd * (43 * U * G + eh * c2.abs() + H * (43 * U * G * H + G * eh) + 34 * U * (G + c1.abs() + H * c2.abs()))
        if ds is not None:
            dx = dx + ds.double()
            e = e + U * dx.abs()
        self.dx = dx
        self.dx_tol = lambda t: EPS[t] * dx.abs() + e * (1 + EPS[t]) + TINY[t]
        # dw, db: rows are added up in a lane, a block and a join: fewer than 64 + rows / 1024 + 1024 / 64 + 16 terms deep
        n = 100 + s.shape[0] / 1024
        self.dw, self.db = (dy * h).sum(0), dy.sum(0)
        self.dw_tol = n * U * (dy * h).abs().sum(0) + (dy.abs() * eh).sum(0) + 1e-37
        self.db_tol = n * U * dy.abs().sum(0) + 1e-37


class LinearRef:
    """y and the gradients of linear_ckpt8 in fp64, with their bounds.

    Operands are rounded to x's type t: w exactly as the kernel does (one cast), act(x) within EPS[t] of its
    value plus SLACK * |x| for the fp32 evaluation of the erf form."""

    SLACK = 8 * U

    def __init__(self, x, w, b, act, dy=None):
        t = x.dtype
        xd, wd = x.detach().double(), w.detach().to(t).double()
        bd = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if b is None else b.detach().double()
        k, n, m = w.shape[1], w.shape[0], x.shape[0]

        def operand(v):
            if act == "none":
                return v, torch.zeros_like(v)
            a = gelu(v)
            return a, (EPS[t] * a.abs() + self.SLACK * v.abs()) * (1 + EPS[t]) + TINY[t]

        a, ea = operand(xd)
        self.y = a @ wd.t() + bd
        e = (k + 2) * U * ((a.abs() + ea) @ wd.abs().t() + bd.abs()) + ea @ wd.abs().t()
        self.y_tol = EPS[t] * self.y.abs() + e * (1 + EPS[t]) + TINY[t]
        if dy is None:
            return
        wt = w.dtype
        dyd, z = dy.double(), checkpoint(x.detach())
        p = dyd @ wd
        e = (n + 2) * U * (dyd.abs() @ wd.abs())
        if act == "gelu":
            slope = gelu_slope(z)
            e = e * slope.abs() + (p.abs() + e) * 2.0 ** -19  # the slope in fp32: erf and exp to a few u, |slope| < 1.13
            p = p * slope
        self.dx = p
        self.dx_tol = EPS[t] * p.abs() + e * (1 + EPS[t]) + TINY[t]
        a, ea = operand(z)
        self.dw = dyd.t() @ a
        e = (m + 2) * U * (dyd.abs().t() @ (a.abs() + ea)) + dyd.abs().t() @ ea
        self.dw_tol = EPS[wt] * self.dw.abs() + e * (1 + EPS[wt]) + TINY[wt]
        self.db = dyd.sum(0)
        self.db_tol = EPS[wt] * self.db.abs() + (m + 2) * U * dyd.abs().sum(0) * (1 + EPS[wt]) + TINY[wt]
