"""Layer norm, 8-bit checkpoints and the checkpointing linear layer on the GPU at the edges of their types and of
their contracts."""
import pytest
import torch

import _token_ops
from _token_ops import LinearRef, NormRef, check
from realtime_semantic_segmentation_pytorch_amd import ops
from realtime_semantic_segmentation_pytorch_amd.models.smp import get_encoder
from realtime_semantic_segmentation_pytorch_amd.ops.ckpt8 import _pack_reference

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEVICE = "cuda"
DTYPES = [F32, BF16, F16]


@pytest.fixture(autouse=True)
def _lib():
    assert ops.load(), "HIP extension must load on the GPU box"


def _rand(*shape, seed=0, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to("cuda", dtype)


# ------------------------------------------------------------------------------- the top of the range

_blocks = _token_ops.checkpoint


def _held(x, dtype=None):
    """The checkpoint's values in fp64: what its blocks round to, and no more than x's type (or ``dtype``) holds."""
    top = torch.finfo(dtype or x.dtype).max
    return _blocks(x).clamp(-top, top)


def _top_rows(rows, c, dtype, top=1.0):
    """Normal values; some rows with one of the largest of the type, or in the last half step below them."""
    x = _rand(rows, c, dtype=dtype)
    big = torch.finfo(dtype).max
    for row, v in ((1, big), (2, -big), (4, big * 0.9945), (5, -big * 0.993), (7, big * 0.99)):
        x[row, (7 * row) % c] = v * top
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [64, 45])
def test_the_largest_values_come_back_finite(dtype, c):
    x = _top_rows(20, c, dtype)
    p = ops.ckpt8_pack(x)
    codes, scales = _pack_reference(x.cpu())
    assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.scales.cpu(), scales)
    v = ops.ckpt8_unpack(p)
    assert torch.isfinite(v).all() and torch.equal(v.double(), _held(x))
    amax = x.double().abs().amax(1, keepdim=True)
    assert ((v.double() - x.double()).abs() <= amax / 127).all()
    for t in DTYPES:  # the values that the checkpoint stands for, rounded once
        assert torch.equal(ops.ckpt8_unpack(p, t), _held(x).to(t))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("m,k,n", [(70, 96, 16), (70, 45, 7), (3000, 64, 256), (700, 320, 64)])
def test_linear_gradients_at_the_largest_values(monkeypatch, dtype, act, m, k, n):
    monkeypatch.setattr(_token_ops, "checkpoint", _held)
    x = _top_rows(m, k, dtype).requires_grad_(True)
    w = _rand(n, k, seed=1, dtype=dtype, scale=2.0 ** -9).requires_grad_(True)
    b = _rand(n, seed=2, dtype=dtype).requires_grad_(True)
    dy = _rand(m, n, seed=3, dtype=dtype, scale=2.0 ** -9)
    dy[1] = 0  # 0 times a finite value
    y = ops.linear_ckpt8(x, w, b, act=act)
    y.backward(dy)
    ref = LinearRef(x, w, b, act, dy)
    check(y, ref.y, ref.y_tol, "y")
    check(x.grad, ref.dx, ref.dx_tol, "dx")
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")


@pytest.mark.parametrize("c", [64, 45, 520, 2056])
def test_layer_norm_gradients_at_the_largest_values(monkeypatch, c):
    monkeypatch.setattr(_token_ops, "checkpoint", lambda s: _held(s, F16))  # NormRef has s in fp64
    x = _top_rows(20, c, F16).requires_grad_(True)  # the variance is a number in fp32
    w, b = (1 + _rand(c, seed=1, scale=0.2)).requires_grad_(True), _rand(c, seed=2).requires_grad_(True)
    dy = _rand(20, c, seed=3, dtype=F16)
    y = ops.layer_norm(x, w, b, ckpt8=True)
    y.backward(dy)
    ref = NormRef(x, w, b, 1e-5, None, F16, dy, None, True)
    check(y, ref.y, ref.y_tol, "y")
    check(x.grad, ref.dx, ref.dx_tol(F16), "dx")
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")
    for t in (F32, BF16):  # it is infinite: rstd = 0, and so is the gradient of that row
        x = _top_rows(20, c, t).requires_grad_(True)
        ops.layer_norm(x, w, b, ckpt8=True).backward(dy.to(t))
        assert torch.isfinite(x.grad).all() and not x.grad[1].any()


# ------------------------------------------------------------------------------- infinities


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [32, 33])
def test_gelu_of_infinities_and_nan_is_the_stock_one(dtype, n):
    """One row each: gelu(-inf) = -inf * 0 is NaN in every type."""
    x = torch.zeros(6, n, device="cuda", dtype=dtype)
    at = torch.tensor([float("-inf"), float("inf"), float("nan"), float("nan"), torch.finfo(dtype).min, torch.finfo(dtype).max])
    x[torch.arange(6), 0] = at.to("cuda", dtype)
    x[3, 0] = -x[3, 0]  # a NaN with its sign set
    w = torch.zeros(n, n, device="cuda", dtype=dtype)
    w[0, 0] = 1.0
    got = ops.linear_ckpt8(x, w, None, act="gelu")[:, 0]
    want = torch.nn.functional.gelu(x[:, 0].float()).to(dtype)
    assert torch.isnan(want[[0, 2, 3]]).all()
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


# ------------------------------------------------------------------------------- hooks of a Mix Transformer


@pytest.mark.parametrize("convert", [ops.convert_layernorm, ops.convert_ckpt8])
@pytest.mark.parametrize("amp", [False, True])
def test_hooks_of_a_mit_see_the_stock_tensors(convert, amp):
    torch.manual_seed(0)
    e, x = get_encoder("mit_b0").cuda().eval(), _rand(1, 3, 64, 64)
    ref, seen = [], []

    def run(into):
        with torch.autocast("cuda", dtype=BF16, enabled=amp):
            hooks = [m.register_forward_hook(lambda m, args, out, n=n: into.append((n, args[0].detach(), out.detach())))
                     for n, m in e.named_modules()
                     if n.count(".") == 1 and n.startswith("block") or n.endswith(("norm1", "norm2", "norm3", "mlp.act", "mlp.fc2"))]
            out = e(x)
            for h in hooks:
                h.remove()
            return out, e(x)

    want = run(ref)
    convert(e)
    got = run(seen)
    assert [n for n, _, _ in seen] == [n for n, _, _ in ref] and "block1.0.mlp.act" in {n for n, _, _ in seen}
    tol = 3e-2 if amp else 1e-4  # bf16 products in another order, 2^-8 a rounding over 8 blocks; fp32 sums in another order
    for a, b in [(p[i], q[i]) for p, q in zip(seen, ref) for i in (1, 2)] + [pq for g, w in zip(got, want) for pq in zip(g, w)]:
        assert a.shape == b.shape and a.dtype == b.dtype
        if a.numel():
            assert float((a.float() - b.float()).norm() / b.float().norm()) < tol


# ------------------------------------------------------------------------------- rows without a variance


@pytest.mark.parametrize("c", [1, 7, 48, 64, 161, 320, 512, 520, 2056, 4101, 8192])
@pytest.mark.parametrize("value", [1000.1, -1000.1, 0.1, 3333.3333, 1e-3])
def test_a_constant_row_has_no_variance(c, value):
    """The mean of equal values is that value: with a mean that is 41 roundings off, 1000.1 would come out as 0.18
    behind eps = 1e-6."""
    b = _rand(c, seed=1)
    for t in (F32, BF16):
        x = torch.full((5, c), value, device="cuda", dtype=t)
        for ckpt in (False, True):
            leaf = x.clone().requires_grad_(True)
            y = ops.layer_norm(leaf, None, b, 1e-6, out_dtype=F32, ckpt8=ckpt)
            assert torch.equal(y, b.expand(5, c))
        assert not ops.layer_norm(x, None, None, 1e-6).any()
        s, y = ops.layer_norm(x, None, None, 1e-6, residual=torch.full_like(x, 3 * value))
        assert not y.any()


@pytest.mark.parametrize("c", [48, 161, 320, 2056])
def test_rows_of_a_large_mean(c):
    """A mean within two roundings of itself, u |mean| each, instead of 41: h is off by 2 u A rstd and rstd's 30 u |h|
    (_token_ops.NormRef), the products and the bias by 3 u |y|."""
    x = _rand(64, c, scale=0.05) + 1000.1
    ref = NormRef(x, None, None, 1e-6)
    s = x.double()
    rstd = 1 / torch.sqrt(s.var(1, correction=0, keepdim=True) + 1e-6)
    u = 2.0 ** -24
    tol = 2 * u * s.abs().amax(1, keepdim=True) * rstd + 33 * u * ref.y.abs()
    check(ops.layer_norm(x, None, None, 1e-6), ref.y, tol, "y")


# ------------------------------------------------------------------------------- tracing and transforms


def _calls():
    m = torch.nn.LayerNorm(32).to(DEVICE).requires_grad_(False)  # a trace holds no constant with a gradient
    ops.convert_layernorm(torch.nn.Sequential(m))
    w, b = _rand(24, 32, seed=1), _rand(24, seed=2)
    yield m, lambda x: torch.nn.functional.layer_norm(x, (32,), m.weight, m.bias, m.eps)
    yield (lambda x: m(x, residual=2 * x)[1]), lambda x: torch.nn.functional.layer_norm(3 * x, (32,), m.weight, m.bias, m.eps)
    yield (lambda x: ops.layer_norm(x, ckpt8=True)), lambda x: torch.nn.functional.layer_norm(x, (32,))
    yield (lambda x: ops.linear_ckpt8(x, w, b, act="gelu")), lambda x: torch.nn.functional.gelu(x) @ w.t() + b


def test_tracing_and_transforms_take_the_stock_operators():
    x, v = _rand(6, 32), _rand(6, 32, seed=3)
    close = dict(rtol=1e-5, atol=1e-5)  # fp32 sums of 32 terms in another order
    for f, ref in _calls():
        torch.testing.assert_close(torch.func.grad(lambda a: f(a).square().sum())(x), torch.func.grad(lambda a: ref(a).square().sum())(x), rtol=1e-4, atol=1e-4)
        torch.testing.assert_close(torch.func.vmap(f)(x), ref(x), **close)
        for got, want in zip(torch.func.jvp(f, (x,), (v,)), torch.func.jvp(ref, (x,), (v,))):
            torch.testing.assert_close(got, want, **close)
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, v)
            got, want = (torch.autograd.forward_ad.unpack_dual(g(dual)).tangent for g in (f, ref))
        torch.testing.assert_close(got, want, **close)
        with torch.no_grad():
            traced = torch.jit.trace(f, (x,), check_trace=False)
        assert "rtseg" not in str(traced.inlined_graph)
        torch.testing.assert_close(traced(v), ref(v), **close)
        with torch._subclasses.FakeTensorMode(allow_non_fake_inputs=True) as mode:
            assert f(mode.from_tensor(x)).shape == ref(x).shape
