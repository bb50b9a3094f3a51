"""Layer norm, 8-bit checkpoints and the checkpointing linear layer on tensors of more than 2^32 elements:
the first and the last rows against 64 bits, zeros between them."""
import pytest
import torch

from _token_ops import LinearRef, NormRef, check
from realtime_semantic_segmentation_pytorch_amd import ops
from realtime_semantic_segmentation_pytorch_amd.ops.ckpt8 import _pack_reference

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
ROWS, C, HEAD, TAIL = 2 ** 26 + 1031, 64, 200, 331  # 2^32 + 65984 elements


@pytest.fixture(autouse=True)
def _lib():
    assert ops.load(), "HIP extension must load"
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB of device memory")
    yield
    torch.cuda.empty_cache()


def _rand(rows, c, seed):
    return torch.randn(rows, c, generator=torch.Generator().manual_seed(seed)).to("cuda", BF16)


def _sparse(small):
    t = torch.zeros(ROWS, C, device="cuda", dtype=BF16)
    t[:HEAD], t[-TAIL:] = small[:HEAD], small[HEAD:]
    return t


def _ends(t):
    return torch.cat([t[:HEAD], t[-TAIL:]])


def _middle(t):
    return t[HEAD:-TAIL]


def test_pack_and_unpack():
    x0 = _rand(HEAD + TAIL, C, 0)
    p = ops.ckpt8_pack(_sparse(x0))
    codes, scales = _pack_reference(x0.cpu())
    assert torch.equal(_ends(p.codes).cpu(), codes) and torch.equal(_ends(p.scales).cpu(), scales)
    assert not _middle(p.codes).any() and bool((_middle(p.scales) == 1).all())
    v = ops.ckpt8_unpack(p)
    del p
    assert torch.equal(_ends(v), ops.ckpt8_unpack(ops.ckpt8_pack(x0))) and not _middle(v).any()


@pytest.mark.parametrize("ckpt", [False, True])
def test_layer_norm(ckpt):
    x0, dy0 = _rand(HEAD + TAIL, C, 0), _rand(HEAD + TAIL, C, 1)
    w, b = (torch.rand(C, generator=torch.Generator().manual_seed(s)).cuda().requires_grad_(True) for s in (2, 3))
    ref = NormRef(x0, w, b, 1e-5, None, BF16, dy0, None, ckpt)
    x = _sparse(x0).requires_grad_(True)
    y = ops.layer_norm(x, w, b, ckpt8=ckpt)
    check(_ends(y), ref.y, ref.y_tol, "y")
    assert bool((_middle(y) == b.to(BF16)).all())
    y.backward(_sparse(dy0))
    check(_ends(x.grad), ref.dx, ref.dx_tol(BF16), "dx")
    assert not _middle(x.grad).any()
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")


def test_linear():
    x0, dy0 = _rand(HEAD + TAIL, C, 0), _rand(HEAD + TAIL, C, 1)
    w, b = (_rand(C, C, 2) / 8).requires_grad_(True), _rand(1, C, 3)[0].requires_grad_(True)
    ref = LinearRef(x0, w, b, "gelu", dy0)
    x = _sparse(x0).requires_grad_(True)
    y = ops.linear_ckpt8(x, w, b, act="gelu")
    check(_ends(y), ref.y, ref.y_tol, "y")
    assert bool((_middle(y) == b).all())
    y.backward(_sparse(dy0))
    check(_ends(x.grad), ref.dx, ref.dx_tol, "dx")
    assert not _middle(x.grad).any()
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")


# ------------------------------------------------------------------------------- more blocks than a launch holds


def _rows(rows, cut):
    return torch.cat([torch.arange(20), torch.arange(cut - 20, cut + 20), torch.arange(rows - 20, rows)]).cuda()


def test_layer_norm_of_more_rows_than_one_launch_holds():
    c, cut = 512, 4 * (2 ** 24 - 1) // 64 * 64  # 4 rows a block
    rows = cut + 777
    if torch.cuda.mem_get_info()[0] < 190 << 30:
        pytest.skip("needs 190 GB of device memory")
    at = _rows(rows, cut)
    x0, dy0 = _rand(len(at), c, 0), _rand(len(at), c, 1)
    w, b = (torch.rand(c, generator=torch.Generator().manual_seed(s)).cuda().requires_grad_(True) for s in (2, 3))
    ref = NormRef(x0, w, b, 1e-5, None, BF16, dy0, None, True)
    x = torch.zeros(rows, c, device="cuda", dtype=BF16)
    x[at] = x0
    y = ops.layer_norm(x, w, b, ckpt8=True)
    del x
    check(y[at], ref.y, ref.y_tol, "y")
    dy = torch.zeros_like(y)
    dy[at] = dy0
    y.backward(dy)
    check(w.grad, ref.dw, ref.dw_tol, "dw")
    check(b.grad, ref.db, ref.db_tol, "db")


@pytest.mark.parametrize("k,n", [(64, 2 ** 20), (2 ** 20, 8)])
def test_linear_of_more_tiles_than_one_launch_holds(k, n):
    cut = (2 ** 24 - 1) // 2 ** 14 * 16
    rows = cut + 777
    at = _rows(rows, cut)
    x0, dy0 = _rand(len(at), k, 0), _rand(len(at), n, 1)
    w = (_rand(n, k, 2) / 8).requires_grad_(True)
    x = torch.zeros(rows, k, device="cuda", dtype=BF16)
    x[at] = x0
    x.requires_grad_(True)
    y = ops.linear_ckpt8(x, w, None, act="gelu")
    dy = torch.zeros_like(y)
    dy[at] = dy0
    y.backward(dy)
    ref = LinearRef(x0, w, None, "gelu", dy0)
    check(y[at], ref.y, ref.y_tol, "y")
    check(x.grad[at], ref.dx, ref.dx_tol, "dx")
    check(w.grad, ref.dw, ref.dw_tol, "dw")
