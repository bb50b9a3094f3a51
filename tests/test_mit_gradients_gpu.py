"""Every parameter gradient of a Mix Transformer encoder on the token operators: against the stock norms in fp32, on
8-bit checkpoints against none, and replayed from a graph against eager steps.  The loss weighs the features with random
numbers, so that no gradient cancels in front of a norm, and every parameter is held to its own gradient."""
import math

import pytest
import torch

from realtime_semantic_segmentation_pytorch_amd import ops
from realtime_semantic_segmentation_pytorch_amd.configs import BaseConfig
from realtime_semantic_segmentation_pytorch_amd.models import get_model

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _lib():
    assert ops.load(), "HIP extension must load on the GPU box"


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _encoder(**kw):
    c = BaseConfig()
    c.model, c.decoder, c.encoder, c.encoder_weights, c.num_class = "smp", "fpn", "mit_b0", None, 5
    for k, v in kw.items():
        setattr(c, k, v)
    torch.manual_seed(0)
    e = get_model(c).encoder.cuda().to(memory_format=torch.channels_last).train()
    for d in e.modules():
        if hasattr(d, "p"):
            d.p = 0.0  # drop path: every variant takes the same path
    with torch.no_grad():  # no symmetry left of the initialisation: zero biases, unit norms, projections of 0.02
        for i, p in enumerate(e.parameters()):
            p.add_(0.1 * p.std().nan_to_num() * _rand(*p.shape, seed=i) + (0.05 * _rand(*p.shape, seed=i) if p.dim() == 1 else 0))
    return e


def _params(e):
    return {n: p for n, p in e.named_parameters() if not n.startswith("head.")}


def _weights(e, x):
    with torch.no_grad():
        return [_rand(*f.shape, seed=50 + i) for i, f in enumerate(e(x)[2:])]


def _grads(e, x, weigh, amp=False):
    params = _params(e)
    with torch.autocast("cuda", dtype=BF16, enabled=amp, cache_enabled=False):
        loss = sum((f.float() * r).mean() for f, r in zip(e(x)[2:], weigh))
    return dict(zip(params, torch.autograd.grad(loss, list(params.values()))))


def _check(got, want, tol):
    """|got - want| <= tol(name) |want|, parameter by parameter; a floor of 2^-20 of the whole gradient."""
    total = float(torch.stack([g.float().norm() for g in want.values()]).norm())
    for n, w in want.items():
        d, own = float((got[n].float() - w.float()).norm()), float(w.float().norm())
        assert d <= tol(n) * own + 2.0 ** -20 * total, (n, d / own, tol(n))


def test_every_gradient_in_fp32_is_that_of_the_stock_norms():
    """A layer's sums have up to 4096 terms: 2^-24 sqrt(4096) of their result where roundings are independent; 64 layers
    in a row, all in one direction, make 2.5e-4."""
    x = _rand(2, 3, 64, 96).contiguous(memory_format=torch.channels_last)
    a, b = _encoder(hip_layernorm=False), _encoder()
    assert any(isinstance(m, ops.LayerNorm) for m in b.modules()) and not any(isinstance(m, ops.LayerNorm) for m in a.modules())
    weigh = _weights(a, x)
    _check(_grads(b, x, weigh), _grads(a, x, weigh), lambda n: 2.5e-4)


def _blocks_behind(name):
    """Blocks from this parameter's own to the last one (2 a stage); those of a stage's norm and embedding alike."""
    stage = int(next(c for c in name if c.isdigit()))
    if name.startswith("norm"):
        return 8 - 2 * stage + 1
    return 8 - 2 * (stage - 1) - (int(name.split(".")[1]) if name.startswith("block") else 0)


@pytest.mark.parametrize("amp", [False, True])
def test_every_gradient_on_checkpoints_is_near_the_one_without(amp):
    """A block's scale is above max / 127 and at most max / 63.5, a value off by its 1 / sqrt(12) in the mean square: with
    a largest of 32 values of up to 3 sigma, 3 / 63.5 / 3.46 = 0.014 of sigma.  Every gradient of a block is computed from
    some of its 6 checkpoints (2 norms, 4 linear layers and convs in a row), the errors are independent, and those of
    the blocks behind add up as squares do; three times that is allowed.  bf16 steps differ by their own roundings too: 2^-9
    a rounding in the mean, 20 a block."""
    x = _rand(2, 3, 128, 128, seed=7).contiguous(memory_format=torch.channels_last)
    a, b = _encoder(), _encoder(act_ckpt8=True)
    weigh = _weights(a, x)

    def tol(n):
        k = _blocks_behind(n)
        return 3 * math.hypot(0.014 * math.sqrt(6 * k), 2.0 ** -9 * math.sqrt(20 * 8) if amp else 0.0)

    got, want = _grads(b, x, weigh, amp), _grads(a, x, weigh, amp)
    assert any(not torch.equal(got[n], want[n]) for n in want)
    _check(got, want, tol)


@pytest.mark.no_guard
@pytest.mark.parametrize("kw", [{}, {"act_ckpt8": True}])
def test_every_gradient_of_a_replayed_step_is_the_eager_one(kw):
    """The library's data gradient of a patch embedding is not the same fp32 bits on every run (1e-7), and where its rounding
    to bf16 falls on the other side an element moves by 2^-8 of itself: 2e-2 is five such roundings in a row, all of them
    and all in one direction."""
    x = _rand(2, 3, 64, 64).contiguous(memory_format=torch.channels_last)
    e = _encoder(**kw)
    weigh = _weights(e, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _grads(e, x, weigh, True)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _grads(e, x, weigh, True)
    for turn in range(4):
        x.copy_(_rand(*x.shape, seed=turn))
        g.replay()
        _check(out, _grads(e, x, weigh, True), lambda n: 2e-2)
        torch.cuda.synchronize()
