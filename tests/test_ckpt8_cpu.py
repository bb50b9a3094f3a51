"""Layer norm, 8-bit activation checkpoints and the checkpointing linear layer on CPU tensors: the format,
the formulas against 64 bits and against differences, the refusals, and the Mix Transformer on them."""
import weakref

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from _token_ops import LinearRef, NormRef, check, checkpoint
from realtime_semantic_segmentation_pytorch_amd import ops
from realtime_semantic_segmentation_pytorch_amd.configs import BaseConfig, load_parser
from realtime_semantic_segmentation_pytorch_amd.models import get_model
from realtime_semantic_segmentation_pytorch_amd.models.smp import get_encoder

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


# ------------------------------------------------------------------------------- the format


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 32), (2, 3, 33), (7, 160), (0, 64), (4, 5, 6, 40)])
def test_pack_unpack_values(dtype, shape):
    x = _rand(*shape, dtype=dtype, scale=3.0)
    p = ops.ckpt8_pack(x)
    c = shape[-1]
    assert p.codes.dtype == torch.int8 and p.codes.shape == (x.numel() // c, (c + 31) // 32 * 32)
    assert p.scales.dtype == torch.uint8 and p.scales.shape == (x.numel() // c, (c + 31) // 32)
    assert not p.codes[:, c:].any()
    got = ops.ckpt8_unpack(p)
    assert got.shape == x.shape and got.dtype == dtype
    ref = checkpoint(x.reshape(-1, c)).view(shape)
    assert torch.equal(got.double(), ref)  # q * 2^e fits every type
    amax = x.double().abs().reshape(-1, c).amax(1) if x.numel() else torch.zeros(0, dtype=torch.float64)
    # half of the scale 2^e, and 127 * 2^(e - 1) < max|x|
    err = (got.double() - x.double()).abs().reshape(-1, c)
    assert (err <= (amax / 127).unsqueeze(1)).all()


def test_scale_edges():
    x = torch.zeros(8, 32)
    x[0, 0] = 127.0           # exactly 127 * 2^0
    x[1, 0] = 127.00001       # one step above: the next scale
    x[2, 0] = -127.0 * 2 ** 20
    x[3, :2] = torch.tensor([127.0, 0.5])   # a tie: to even
    x[4, :2] = torch.tensor([127.0, 1.5])
    x[5, 0] = 2.0 ** -140     # below the smallest scale: 0
    x[6, 0] = torch.finfo(torch.float32).max
    p = ops.ckpt8_pack(x)
    assert p.scales[:, 0].tolist() == [127, 128, 147, 127, 127, 1, 249, 1]
    assert p.codes[0, 0] == 127 and p.codes[1, 0] == 64 and p.codes[2, 0] == -127
    assert p.codes[3, 1] == 0 and p.codes[4, 1] == 2 and not p.codes[5].any() and not p.codes[7].any()
    v = ops.ckpt8_unpack(p)
    assert torch.equal(v[2], x[2]) and torch.equal(v[7], x[7]) and v[5, 0] == 0


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_non_finite_block_comes_back_as_nan(bad):
    x = _rand(3, 96)
    x[1, 40] = bad
    p = ops.ckpt8_pack(x)
    assert p.scales[1, 1] == 255 and not p.codes[1, 32:64].any()
    v = ops.ckpt8_unpack(p)
    assert torch.isnan(v[1, 32:64]).all() and torch.isfinite(v[1, :32]).all() and torch.isfinite(v[1, 64:]).all()
    assert torch.isfinite(v[0]).all() and torch.isfinite(v[2]).all()


def test_pack_takes_strided_inputs_and_other_unpack_types():
    x = _rand(6, 80)
    assert torch.equal(ops.ckpt8_pack(x.t()).codes, ops.ckpt8_pack(x.t().contiguous()).codes)
    assert torch.equal(ops.ckpt8_unpack(ops.ckpt8_pack(x), torch.bfloat16).float(), ops.ckpt8_unpack(ops.ckpt8_pack(x)))


def test_ckpt8_saved_holds_one_tensor():
    conv = nn.Conv2d(8, 8, 3, padding=1, groups=8)
    x = _rand(2, 8, 5, 6).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    with ops.ckpt8_saved(x):
        y = conv(x)
    y.backward(_rand(*y.shape, seed=1))
    z = ops.ckpt8_unpack(ops.ckpt8_pack(x.detach().permute(0, 2, 3, 1))).permute(0, 3, 1, 2).contiguous()
    ref = nn.Conv2d(8, 8, 3, padding=1, groups=8)
    ref.load_state_dict(conv.state_dict())
    zr = z.clone().requires_grad_(True)
    ref(zr).backward(_rand(*y.shape, seed=1))
    torch.testing.assert_close(conv.weight.grad, ref.weight.grad, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(x.grad, zr.grad, rtol=1e-6, atol=1e-6)
    with ops.ckpt8_saved(None):
        pass


def test_ckpt8_saved_lets_the_tensor_go():
    w = _rand(8, 1, 3, 3).requires_grad_(True)
    x = (_rand(2, 8, 5, 6).requires_grad_(True) * 2).contiguous(memory_format=torch.channels_last)
    gone = weakref.ref(x)
    with ops.ckpt8_saved(x):
        y = F.conv2d(x, w, None, 1, 1, 1, 8)
    del x
    assert gone() is None and y.requires_grad


# ------------------------------------------------------------------------------- linear


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (5, 33, 7), (9, 64, 40), (0, 8, 4)])
def test_linear_against_64_bits(dtype, act, m, k, n):
    x = _rand(m, k, dtype=dtype, scale=2.0).requires_grad_(True)
    w = _rand(n, k, seed=1, dtype=dtype, scale=k ** -0.5).requires_grad_(True)
    b = _rand(n, seed=2, dtype=dtype).requires_grad_(True)
    dy = _rand(m, n, seed=3, dtype=dtype)
    y = ops.linear_ckpt8(x, w, b, act=act)
    y.backward(dy)
    ref = LinearRef(x, w, b, act, dy)
    check(y, ref.y, ref.y_tol, "y")
    check(x.grad, ref.dx, ref.dx_tol, "dx")
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")


@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_gradient_against_differences(act):
    """At inputs that their own checkpoint holds exactly the gradients are those of the function itself."""
    x = (torch.randint(-127, 128, (4, 40), generator=torch.Generator().manual_seed(0)) / 64.0)
    x[:, 0], x[:, 32] = 127 / 64.0, -127 / 64.0
    assert torch.equal(ops.ckpt8_unpack(ops.ckpt8_pack(x)), x)
    w, b, dy = _rand(3, 40, seed=1), _rand(3, seed=2), _rand(4, 3, seed=3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ops.linear_ckpt8(*leaves, act=act).backward(dy)

    def f(x, w, b):
        a = F.gelu(x) if act == "gelu" else x
        return float(((a @ w.t() + b) * dy.double()).sum())

    h = 1e-5
    base = [t.double() for t in (x, w, b)]
    for which, leaf in enumerate(leaves):
        for i in (0, 1, leaf.numel() // 2, leaf.numel() - 1):
            vals = []
            for sign in (1, -1):
                args = [t.clone() for t in base]
                args[which].view(-1)[i] += sign * h
                vals.append(f(*args))
            # central differences: h^2 / 6 times a third derivative of a few units, and the fp32 sums of 40 terms
            assert abs((vals[0] - vals[1]) / (2 * h) - float(leaf.grad.view(-1)[i])) < 2e-5


def test_linear_keeps_codes_alone():
    x = _rand(64, 96, dtype=torch.bfloat16).requires_grad_(True)
    w = _rand(32, 96, seed=1, dtype=torch.bfloat16).requires_grad_(True)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        y = ops.linear_ckpt8(x, w, None, act="gelu")
    assert y.requires_grad
    assert sum(t.numel() * t.element_size() for t in held if t.data_ptr() != w.data_ptr()) == 64 * 96 + 64 * 3
    held.clear()
    with torch.no_grad(), torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        assert torch.equal(ops.linear_ckpt8(x, w, None, act="gelu"), y)
    assert not held


@pytest.mark.parametrize("frozen", ["x", "w", "b", "xw", "wb"])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_partial_gradients(frozen, act):
    leaves = {"x": _rand(6, 40), "w": _rand(5, 40, seed=1), "b": _rand(5, seed=2)}
    full = {k: v.clone().requires_grad_(True) for k, v in leaves.items()}
    part = {k: v.clone().requires_grad_(k not in frozen) for k, v in leaves.items()}
    for d in (full, part):
        ops.linear_ckpt8(d["x"], d["w"], d["b"], act=act).square().sum().backward()
    for k in leaves:
        assert part[k].grad is None if k in frozen else torch.equal(part[k].grad, full[k].grad)


def test_linear_master_weights_and_autocast():
    x = _rand(3, 5, 48, dtype=torch.bfloat16).requires_grad_(True)
    w, b = _rand(7, 48, seed=1).requires_grad_(True), _rand(7, seed=2).requires_grad_(True)
    y = ops.linear_ckpt8(x, w, b)
    assert y.shape == (3, 5, 7) and y.dtype == torch.bfloat16
    y.sum().backward()
    assert w.grad.dtype == torch.float32 and b.grad.dtype == torch.float32 and x.grad.dtype == torch.bfloat16
    with torch.autocast("cpu", dtype=torch.bfloat16):
        z = ops.linear_ckpt8(x.float(), w, b)
    assert z.dtype == torch.bfloat16 and torch.equal(z, y)


def test_linear_refusals():
    x, w, b = _rand(4, 8), _rand(3, 8), _rand(3)
    with pytest.raises(ValueError, match="act must be one of"):
        ops.linear_ckpt8(x, w, b, act="relu")
    with pytest.raises(ValueError, match="weight must be"):
        ops.linear_ckpt8(x, _rand(3, 9), b)
    with pytest.raises(ValueError, match="weight must be"):
        ops.linear_ckpt8(x, _rand(8), b)
    with pytest.raises(ValueError, match="weight must be"):
        ops.linear_ckpt8(x, _rand(0, 8), None)
    with pytest.raises(ValueError, match="bias must have"):
        ops.linear_ckpt8(x, w, _rand(4))
    with pytest.raises(TypeError, match="of one type"):
        ops.linear_ckpt8(x, w, b.bfloat16())
    with pytest.raises(TypeError, match="x's type"):
        ops.linear_ckpt8(x, w.bfloat16(), None)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        ops.linear_ckpt8(x.double(), w.double(), None)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        ops.ckpt8_pack(torch.zeros(4, 8, dtype=torch.int32))
    with pytest.raises(ValueError, match="at least one channel"):
        ops.ckpt8_pack(torch.zeros(4, 0))
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        ops.ckpt8_unpack(ops.ckpt8_pack(x), torch.int8)
    y = ops.linear_ckpt8(x.requires_grad_(True), w.requires_grad_(True), None)
    (g,) = torch.autograd.grad(y.sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g * w).sum().backward()


# ------------------------------------------------------------------------------- layer norm


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,c", [(1, 1), (4, 33), (7, 64), (0, 16)])
def test_layer_norm_against_64_bits(rows, c, residual, ckpt):
    x = _rand(rows, c).requires_grad_(True)
    r = _rand(rows, c, seed=1).requires_grad_(True) if residual else None
    w, b = (1 + 0.1 * _rand(c, seed=2)).requires_grad_(True), _rand(c, seed=3).requires_grad_(True)
    dy, ds = _rand(rows, c, seed=4), _rand(rows, c, seed=5)
    got = ops.layer_norm(x, w, b, 1e-5, residual=r, ckpt8=ckpt)
    ref = NormRef(x, w, b, 1e-5, r, dy=dy, ds=ds if residual else None, ckpt=ckpt)
    if residual:
        torch.autograd.backward(got, (ds, dy))
        assert torch.equal(got[0].double(), ref.s)
        check(r.grad, ref.dx, ref.dx_tol(torch.float32), "dres")
        y = got[1]
    else:
        got.backward(dy)
        y = got
    check(y, ref.y, ref.y_tol, "y")
    check(x.grad, ref.dx, ref.dx_tol(torch.float32), "dx")
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")


def test_layer_norm_types_and_refusals():
    x = _rand(4, 8, dtype=torch.bfloat16)
    assert ops.layer_norm(x).dtype == torch.bfloat16
    assert ops.layer_norm(x, out_dtype=torch.float32).dtype == torch.float32
    s, y = ops.layer_norm(x.float(), residual=x)
    assert s.dtype == y.dtype == torch.float32
    s, y = ops.layer_norm(x, residual=x.float(), want_sum=False)
    assert s is None and y.dtype == torch.float32
    with pytest.raises(ValueError, match="weight must have"):
        ops.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="residual must have"):
        ops.layer_norm(x, residual=x[:3])
    with pytest.raises(ValueError, match="at least one channel"):
        ops.layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="floating"):
        ops.layer_norm(x, out_dtype=torch.int8)


def test_layer_norm_module_keeps_the_stock_result_and_keys():
    m = nn.Sequential(nn.LayerNorm(24, eps=1e-6), nn.LayerNorm((4, 24)), nn.LayerNorm(24, elementwise_affine=False))
    keys, x = list(m.state_dict()), _rand(3, 4, 24)
    ref = m(x)
    ops.convert_layernorm(m)
    assert all(type(c) is ops.LayerNorm for c in m) and list(m.state_dict()) == keys
    assert torch.equal(m(x), ref)
    with pytest.raises(ValueError, match="last axis alone"):
        m[1](x, residual=x)
    with pytest.raises(ValueError, match="channels expected"):
        m[0](x[..., :7])


# ------------------------------------------------------------------------------- the models


def _config(**kw):
    c = BaseConfig()
    c.model, c.decoder, c.encoder, c.encoder_weights, c.num_class = "smp", "fpn", "mit_b0", None, 5
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_mit_is_unchanged_without_checkpoints():
    torch.manual_seed(0)
    e = get_encoder("mit_b0").eval()
    x = _rand(2, 3, 64, 96)
    ref = e(x)
    got = ops.convert_layernorm(e)(x)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_mit_trains_on_checkpoints():
    """Same value, gradients within the checkpoints' error of the stock ones, keys unchanged, the flag parsed."""
    assert load_parser(BaseConfig(), ["--act_ckpt8"]).act_ckpt8 and not BaseConfig().act_ckpt8
    torch.manual_seed(0)
    a = get_model(_config()).train()
    torch.manual_seed(0)
    b = get_model(_config(act_ckpt8=True)).train()
    assert list(a.state_dict()) == list(b.state_dict())
    assert any(isinstance(m, ops.Ckpt8Linear) for m in b.modules()) and not any(isinstance(m, ops.Ckpt8Linear) for m in a.modules())
    x = _rand(2, 3, 64, 64)
    out = []
    for m in (a, b):
        for d in m.modules():
            if hasattr(d, "p"):
                d.p = 0.0  # drop path / dropout: both models take the same path
        y = m(x)
        y.square().mean().backward()
        out.append(y.detach())
    torch.testing.assert_close(out[1], out[0], rtol=1e-4, atol=1e-4)
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        assert (p.grad is None) == (q.grad is None), name
    # the last stage's linear layers, straight behind the loss: one checkpoint's error (at most 1 / 127 of a block's maximum)
    p, q = (m.encoder.block4[1].mlp.fc2.weight.grad for m in (a, b))
    assert float((p - q).norm() / p.norm()) < 2 / 127
