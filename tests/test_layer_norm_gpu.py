"""Layer norm kernels (layer_norm_*.hip via ops.layer_norm) against 64 bits: values, the residual sum, the
gradients, the 8-bit checkpoint form; widths from one channel to the largest, unaligned and strided inputs,
streams and captured graphs."""
import pytest
import torch
import torch.nn as nn

from _token_ops import NormRef, check
from realtime_semantic_segmentation_pytorch_amd import ops

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _lib():
    assert ops.load(), "HIP extension must load on the GPU box"


def _rand(*shape, seed=0, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale + shift).to("cuda", dtype)


def _run(rows, c, x_t, r_t, out_t, ckpt, shift=0.0, affine=True):
    x = _rand(rows, c, dtype=x_t, scale=2.0, shift=shift).requires_grad_(True)
    r = _rand(rows, c, seed=1, dtype=r_t).requires_grad_(True) if r_t is not None else None
    w = (1 + 0.2 * _rand(c, seed=2)).requires_grad_(True) if affine else None
    b = _rand(c, seed=3).requires_grad_(True) if affine else None
    got = ops.layer_norm(x, w, b, 1e-5, residual=r, out_dtype=out_t, ckpt8=ckpt)
    s, y = got if r is not None else (None, got)
    st = x_t if r_t is None else torch.promote_types(x_t, r_t)
    out_t = out_t or st
    assert y.dtype == out_t
    dy = _rand(rows, c, seed=4, dtype=out_t)
    ds = _rand(rows, c, seed=5, dtype=st) if r is not None else None
    ref = NormRef(x, w, b, 1e-5, r, out_t, dy, ds, ckpt)
    torch.autograd.backward([y] if r is None else [s, y], [dy] if r is None else [ds, dy])
    check(y, ref.y, ref.y_tol, "y")
    check(x.grad, ref.dx, ref.dx_tol(x_t), "dx")
    if r is not None:
        assert s.dtype == st and torch.equal(s.double(), ref.s)
        check(r.grad, ref.dx, ref.dx_tol(r_t), "dres")
    if affine:
        check(w.grad, ref.dw, ref.dw_tol, "dw")
        check(b.grad, ref.db, ref.db_tol, "db")


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("c", [1, 7, 8, 31, 32, 33, 64, 96, 160, 161, 256, 320, 512, 520, 1000, 2048, 2056, 4104, 6001, 8192])
def test_widths(c, ckpt):
    _run(37, c, F32, None, None, ckpt)
    _run(5, c, BF16, BF16, None, ckpt)


@pytest.mark.parametrize("rows", [0, 1, 2, 15, 16, 17, 63, 64, 65, 1000, 20011])
@pytest.mark.parametrize("c", [32, 160])
def test_row_counts(rows, c):
    _run(rows, c, F32, BF16, BF16, False)
    _run(rows, c, F16, None, None, True)


@pytest.mark.parametrize("x_t,r_t,out_t", [
    (F32, None, BF16), (F32, None, F16), (F32, F32, F32), (F32, BF16, BF16), (F32, F16, F16), (F32, F16, BF16),
    (BF16, None, F32), (BF16, BF16, F32), (BF16, F32, BF16), (F16, F16, F16), (F16, None, F32), (BF16, F16, F32),
    (BF16, None, F16)])
@pytest.mark.parametrize("c", [40, 45])
def test_types(x_t, r_t, out_t, c):
    if out_t == F16 and x_t == BF16:  # through fp32: two roundings, in the bound of a bf16 one
        x = _rand(9, c, dtype=x_t)
        y = ops.layer_norm(x, out_dtype=out_t)
        assert y.dtype == F16 and torch.equal(y, ops.layer_norm(x, out_dtype=F32).to(F16))
        return
    _run(33, c, x_t, r_t, out_t, False)
    _run(33, c, x_t, r_t, out_t, True)


def test_no_affine_large_mean_and_constant_rows():
    _run(50, 64, F32, None, None, False, affine=False)
    _run(50, 320, F32, None, None, False, shift=1000.0)
    x = torch.full((3, 48), 5.25, device="cuda").requires_grad_(True)
    y = ops.layer_norm(x, eps=1e-6)
    y.sum().backward()
    assert not y.any() and torch.isfinite(x.grad).all()


@pytest.mark.parametrize("c", [3, 45, 161, 2053, 4101])
def test_no_affine_unaligned(c):
    for ckpt in (False, True):
        _run(13, c, F32, None, None, ckpt, affine=False)
        _run(13, c, BF16, BF16, None, ckpt, affine=False)


def test_leaves_of_one_type_keep_gradients_of_their_own():
    x, r = (_rand(6, 32, seed=i).requires_grad_(True) for i in (1, 2))
    for n in (1, 2):  # the second pass adds to what the first one left
        s, y = ops.layer_norm(x, residual=r)
        torch.autograd.backward([s, y], [torch.ones_like(s), _rand(6, 32, seed=3)])
        if n == 1:
            first = x.grad.clone()
        assert torch.equal(x.grad, n * first) and torch.equal(r.grad, n * first)
    assert x.grad.data_ptr() != r.grad.data_ptr()


@pytest.mark.parametrize("shape", [(6, 32), (2, 3, 32)])
def test_a_change_in_place_is_noticed(shape):
    x = _rand(6, 32).view(shape).requires_grad_(True)
    for ckpt in (False, True):
        a = x * 1
        y = ops.layer_norm(a, ckpt8=ckpt)
        b = x * 1
        s, z = ops.layer_norm(x, residual=b, ckpt8=ckpt)
        a.add_(1)
        s.add_(1)
        for t in (y, z):
            if ckpt:  # the checkpoint is of the values at the time
                t.sum().backward()
            else:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    t.sum().backward()


def test_rows_do_not_mix():
    x = _rand(9, 96)
    clean = ops.layer_norm(x)
    x[4, 10], x[6, 0] = float("nan"), float("inf")
    y = ops.layer_norm(x)
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[4]).all() and torch.isnan(y[6]).any()


@pytest.mark.parametrize("ckpt", [False, True])
def test_strided_and_unaligned(ckpt):
    base = _rand(12, 200)
    flat = _rand(1 + 12 * 64, seed=1)
    for x in (base[:, 3:67], base.t()[:64].t(), flat[1:].view(12, 64), base.view(3, 4, 200)[:, :, :64].transpose(0, 1)):
        a = x.detach().requires_grad_(True)
        d = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
        dy = _rand(*x.shape[::-1], seed=2).permute(*range(x.dim() - 1, -1, -1))
        ya, yd = ops.layer_norm(a, ckpt8=ckpt), ops.layer_norm(d, ckpt8=ckpt)
        ya.backward(dy)
        yd.backward(dy.contiguous())
        torch.testing.assert_close(ya, yd, rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(a.grad, d.grad, rtol=1e-5, atol=1e-5)


def test_unused_outputs_and_partial_gradients():
    x, r = _rand(8, 64).requires_grad_(True), _rand(8, 64, seed=1, dtype=BF16).requires_grad_(True)
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    s, y = ops.layer_norm(x, w, b, residual=r)
    s.backward(torch.ones_like(s))  # the norm itself unused
    assert torch.equal(x.grad, torch.ones_like(s)) and torch.equal(r.grad, torch.ones_like(r)) and w.grad is None
    x.grad = r.grad = None
    none, y = ops.layer_norm(x, w, b, residual=r, want_sum=False)
    assert none is None
    y.backward(_rand(8, 64, seed=2))
    gx, gr, gw, gb = x.grad.clone(), r.grad.clone(), w.grad.clone(), b.grad.clone()
    assert torch.equal(gr, gx.to(BF16))
    for keep in ("x", "r", "w", "b"):
        t = {"x": x.detach(), "r": r.detach(), "w": w.detach(), "b": b.detach()}
        t[keep] = t[keep].clone().requires_grad_(True)
        _, y = ops.layer_norm(t["x"], t["w"], t["b"], residual=t["r"])
        y.backward(_rand(8, 64, seed=2))
        assert torch.equal(t[keep].grad, {"x": gx, "r": gr, "w": gw, "b": gb}[keep])


def test_bits_are_the_same_on_every_run_and_stream():
    x, r = _rand(30000, 96).requires_grad_(True), _rand(30000, 96, seed=1, dtype=BF16).requires_grad_(True)
    w, b = _rand(96, seed=2).requires_grad_(True), _rand(96, seed=3).requires_grad_(True)
    dy = _rand(30000, 96, seed=4, dtype=BF16)

    def step():
        s, y = ops.layer_norm(x, w, b, residual=r, out_dtype=BF16)
        return (s.detach(), y.detach(), *torch.autograd.grad((s, y), (x, r, w, b), (s.detach(), dy)))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, second))


@pytest.mark.no_guard
def test_captured_graphs():
    """Two captured training steps, replayed in turn with new inputs and eager work in between."""
    ins, graphs = [], []

    def step(x, w, b, dy, ckpt):
        y = ops.layer_norm(x, w, b, ckpt8=ckpt)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

    for i, (rows, c) in enumerate(((700, 64), (41, 320))):
        t = [_rand(rows, c, seed=i).requires_grad_(True), _rand(c, seed=10).requires_grad_(True),
             _rand(c, seed=11).requires_grad_(True), _rand(rows, c, seed=12)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*t, i == 1)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*t, i == 1)
        ins.append(t)
        graphs.append((g, out))
    for turn in range(4):
        for t in ins:
            with torch.no_grad():
                t[0].copy_(_rand(*t[0].shape, seed=100 + turn))
        for g, _ in graphs:
            g.replay()
        for i, (t, (_, out)) in enumerate(zip(ins, graphs)):
            assert all(torch.equal(a, b) for a, b in zip(out, step(*t, i == 1)))
        torch.cuda.synchronize()


def test_autocast_follows_the_stock_op():
    x = _rand(4, 10, 32, dtype=BF16)
    m = nn.LayerNorm(32).cuda()
    with torch.autocast("cuda", dtype=BF16):
        ref = m(x)
        got = ops.convert_layernorm(nn.Sequential(m))(x)
    assert got.dtype == ref.dtype == F32
    torch.testing.assert_close(got, ref, rtol=1e-5, atol=1e-5)


def test_takes_the_hip_path_and_refuses():
    x = _rand(4, 32).requires_grad_(True)
    assert "LayerNormFn" in ops.layer_norm(x).grad_fn.name()
    wide = _rand(2, 8200)
    torch.testing.assert_close(ops.layer_norm(wide), torch.nn.functional.layer_norm(wide, (8200,)))
    with pytest.raises(RuntimeError):  # on another device
        ops.layer_norm(x, torch.ones(32))
    y = ops.layer_norm(x)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g * x).sum().backward()
    s = ops.layer_norm(x.detach().requires_grad_(True), residual=_rand(4, 32, seed=1))
    with torch.no_grad():
        s[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s[1].sum().backward()
