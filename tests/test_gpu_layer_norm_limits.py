"""LayerNorm at the limits of its rows and values, against the formula in 64 bits under the bounds of test_gpu_block_ops.py."""
import pytest
import torch
from test_gpu_block_ops import DEV, E32, TYPES, _near, _norm_check, _rand, _u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D", [("fp32", 8188), ("fp32", 8192), ("bf16", 16376), ("bf16", 16384)])
@pytest.mark.parametrize("start", [0, 1])
def test_layer_norm_widest_rows(dtype, D, start):
    """The widest rows of whole 16-byte granules run on the kernels, wherever rows and weights start."""
    from torchllmtuner_b200 import ops
    from torchllmtuner_b200.ops.cuda_ext import load
    dt = TYPES[dtype]
    x = _rand(5, D + 24, seed=1, dtype=dt, mean=0.5)[:, start:start + D].detach().requires_grad_()
    wb = _rand(2, D + 8, seed=2, dtype=dt, mean=1, std=0.1)
    w, b = (wb[i, start:start + D].detach().requires_grad_() for i in (0, 1))
    dy = _rand(5, D + 8, seed=4, dtype=dt)[:, start:start + D]
    before = load().launch_count()
    y = ops.layer_norm(x, w, b, 1e-6)
    assert load().launch_count() == before + 1
    grads = torch.autograd.grad(y, (x, w, b), dy)
    assert load().launch_count() == before + 3
    _norm_check(x.detach(), w.detach(), b.detach(), dy, y.detach(), *grads, 1e-6)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_layer_norm_of_tiny_values_without_eps(dtype):
    """Values of 2e-20 and eps 0: 1 / std is 5e19, whose square is beyond fp32. The squares are subnormal (4e-40, held to 2^-18 of themselves), so the
    reciprocal is off by less than 2^-16 of itself; 2^-12 leaves room for the sums."""
    from torchllmtuner_b200 import ops
    dt = TYPES[dtype]
    for D in (64, 200, 1152, 4096):
        x, dy = (_rand(7, D, seed=1) * 2e-20).to(dt).requires_grad_(), _rand(7, D, seed=2, dtype=dt)
        w, b = _rand(D, seed=3, dtype=dt, mean=1, std=0.1).requires_grad_(), _rand(D, seed=4, dtype=dt).requires_grad_()
        y = ops.layer_norm(x, w, b, 0.0)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        X, G, W = x.detach().double(), dy.double(), w.detach().double()
        r = (X - X.mean(1, keepdim=True)).square().mean(1, keepdim=True).rsqrt()
        h, g = (X - X.mean(1, keepdim=True)) * r, G * W
        assert r.max() > 2e19
        _near(y.detach(), h * W + b.detach().double(), _u(dt) * (h * W + b.detach().double()).abs() + 2.0 ** -12 * (h * W).abs() + 1e-6, "y")
        ref = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        _near(dx, ref, _u(dt) * ref.abs() + 2.0 ** -12 * r * (g.abs() + g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True)), "dx")
        _near(dw, (G * h).sum(0), _u(dt) * (G * h).sum(0).abs() + 2.0 ** -12 * (G * h).abs().sum(0) + 1e-6, "dw")
        _near(db, G.sum(0), _u(dt) * G.sum(0).abs() + 128 * E32 * G.abs().sum(0), "db")


def test_layer_norm_of_the_most_rows():
    """2^31 - 1 rows of one column: without a spread y is the bias; the bias's gradient counts the rows."""
    from torchllmtuner_b200 import ops
    R = (1 << 31) - 1
    x = torch.zeros(R, 1, device=DEV, dtype=torch.bfloat16)
    x[-300:] = 3.0
    x.requires_grad_()
    w, b = torch.ones(1, device=DEV, dtype=torch.bfloat16).requires_grad_(), torch.full((1,), 0.75, device=DEV, dtype=torch.bfloat16).requires_grad_()
    y = ops.layer_norm(x, w, b, 1e-6)
    assert (y == 0.75).all()
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    del y
    assert (dx[-1000:].abs() <= 1e-2).all() and dw.abs() <= 3 * 300 * 1000 * 2.0 ** -22      # h is off by a few steps of fp32 of 3 / sqrt(eps)
    assert abs(db.double().item() - R) <= R * 2.0 ** -8
    del x, dx
    torch.cuda.empty_cache()
