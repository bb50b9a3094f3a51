"""The token operators on the GPU against 64 bits at sizes that reach every tile of the checkpointing linear layer's
three kernels (csrc/kernels/linear_ckpt8_*.hip) and every layout of a row in the layer norm's, in every type."""
import pytest
import torch

from _token_ops import LinearRef, check
from test_layer_norm_gpu import _run as run_norm
from realtime_semantic_segmentation_pytorch_amd import ops

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _lib():
    assert ops.load(), "HIP extension must load on the GPU box"


def _rand(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# rows, k, n.  Forward and data gradient choose by ceil(rows / 64) * ceil(width / 256) >= 256, the data gradient also by
# ceil(rows / 64) * ceil(k / 128) >= 256 (mid), and both by the width (n and k) and by whether the sum fits one step (k
# and n <= 64 in 16 bits, 32 in fp32); the weight gradient by n alone.
SIZES = [
    (16411, 64, 256),    # forward: 256 columns, one step (16 bits), k split otherwise; data gradient 64 columns
    (16411, 96, 256),    # forward: 256 columns, looping
    (16411, 32, 200),    # one step in fp32 too, ragged columns
    (16411, 32, 48),     # forward and data gradient: 64 columns, one step
    (16411, 256, 64),    # forward: 64 columns, looping; data gradient: 256 columns, one step (16 bits)
    (16411, 256, 32),    # ... and in fp32
    (16411, 128, 128),   # forward and data gradient: 128 columns, looping
    (16411, 64, 128),    # data gradient: 64 columns, looping
    (16411, 128, 56),    # data gradient: 128 columns, one step
    (8300, 128, 320),    # forward: the 320-column tile behind gelu; weight gradient: 320 columns
    (8300, 136, 264),    # ... ragged
    (16411, 72, 512),    # forward: 512 columns (8 waves) behind gelu; weight gradient: 512 columns
    (16411, 64, 400),    # ... ragged, one step of k
    (4200, 512, 1032),   # two column tiles of 512 and one ragged
    (16411, 320, 160),   # data gradient: 256 columns, looping
    (4200, 512, 512),    # data gradient: 64 x 128 tiles
    (4200, 488, 200),    # ... ragged
    (16411, 257, 161),   # nothing aligned: the large unaligned tiles
    (16411, 33, 515),    # ... of the weight gradient's widest
    (8300, 129, 300),    # ... its 320 columns
    (16411, 31, 97),     # ... its 128 columns
    (16411, 45, 63),     # ... its 64 columns
    (16411, 64, 24),     # fp32, one step: data gradient 64 columns
    (16411, 128, 24),    # ... 128 columns
    (16411, 32, 104),    # ... forward 128 columns
    (16411, 64, 257),    # aligned k, unaligned n: aligned forward, the others not
    (16411, 257, 64),    # unaligned k, aligned n
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_tiles(dtype, act, m, k, n):
    x = _rand(m, k, dtype=dtype, scale=1.5).requires_grad_(True)
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


@pytest.mark.parametrize("x_t", [BF16, F16])
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("m,k,n", [(16411, 64, 256), (16411, 256, 64), (8300, 128, 320), (16411, 257, 161)])
def test_linear_tiles_under_master_weights(x_t, act, m, k, n):
    """fp32 weights, as autocast training holds them: their gradients come in fp32."""
    x = _rand(m, k, dtype=x_t, scale=1.5).requires_grad_(True)
    w, b = _rand(n, k, seed=1, scale=k ** -0.5).requires_grad_(True), _rand(n, seed=2).requires_grad_(True)
    dy = _rand(m, n, seed=3, dtype=x_t)
    y = ops.linear_ckpt8(x, w, b, act=act)
    y.backward(dy)
    ref = LinearRef(x, w, b, act, dy)
    assert w.grad.dtype == b.grad.dtype == F32
    check(y, ref.y, ref.y_tol, "y")
    check(x.grad, ref.dx, ref.dx_tol, "dx")
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", [(1, 1), (63, 65), (4099, 161), (70000, 64)])
def test_bias_gradient_alone(dtype, m, n):
    x, w, dy = _rand(m, 32, dtype=dtype), _rand(n, 32, seed=1, dtype=dtype), _rand(m, n, seed=3, dtype=dtype)
    b = _rand(n, seed=2, dtype=dtype).requires_grad_(True)
    ops.linear_ckpt8(x, w, b).backward(dy)
    ref = LinearRef(x, w, b, "none", dy)
    check(b.grad, ref.db, ref.db_tol, "db")


@pytest.mark.parametrize("x_t,r_t,out_t", [(F32, None, F32), (F32, BF16, BF16), (F32, F16, F16), (BF16, None, F32), (BF16, BF16, BF16),
                                           (F16, None, F32), (F16, F16, F16)])
@pytest.mark.parametrize("c", [40, 45, 64, 320, 161, 1024, 1001, 2016, 1999, 2056, 2053, 4104, 4101])
def test_norm_layouts(x_t, r_t, out_t, c):
    """1 .. 4 vectors of 8 channels a lane, a wave's lanes or a block's, aligned and not."""
    for ckpt in (False, True):
        run_norm(21, c, x_t, r_t, out_t, ckpt)
