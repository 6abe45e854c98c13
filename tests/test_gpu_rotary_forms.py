"""Rotary positions and per-head norms in forms that test_gpu_block_ops.py does not reach, against the formulas in 64 bits under its bounds."""
import math

import pytest
import torch
from test_gpu_block_ops import DEV, E32, _near, _rand, _tables, _turn64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", ["both", "none", "keys"])
@pytest.mark.parametrize("T,H,K,d,P", [(50, 4, 2, 64, 32), (300, 8, 1, 128, 64), (20, 3, 3, 72, 36), (33, 2, 1, 256, 16)])
def test_default_norm_and_rotation_in_fp32_is_the_kernel(T, H, K, d, P, weights):
    from torchllmtuner_b200 import ops
    from torchllmtuner_b200.ops.cuda_ext import load
    cos, sin = _tables(T, P)
    q, k = _rand(T, H, d, seed=1, dtype=torch.float32).requires_grad_(), _rand(T, K, d, seed=2, dtype=torch.float32).requires_grad_()
    qw, kw = (_rand(d, seed=s, dtype=torch.float32, mean=1.0, std=0.1).requires_grad_() for s in (3, 4))
    qw, kw = qw if weights == "both" else None, kw if weights != "none" else None
    dq, dk = _rand(T, H, d, seed=5, dtype=torch.float32), _rand(T, K, d, seed=6, dtype=torch.float32)
    before = load().launch_count()
    yq, yk = ops.qk_norm_rope(q, k, qw, kw, cos, sin, 1e-6)
    assert load().launch_count() > before
    for x, y, w, dy in ((q, yq, qw, dq), (k, yk, kw, dk)):
        X, G = x.detach().double(), dy.double()
        W = w.detach().double() if w is not None else torch.ones(d, device=DEV, dtype=torch.float64)
        r = (X.square().mean(-1, keepdim=True) + 1e-6).rsqrt() if w is not None else torch.ones_like(X[..., :1])
        ref, _ = _turn64(X * r * W, cos, sin, "half", 0)
        size = _turn64((X * r * W).abs(), cos.abs(), -sin.abs(), "half", 0)[1]
        _near(y.detach(), ref, E32 * ref.abs() + 64 * E32 * size, "forward")
        dx, *dw = torch.autograd.grad(y, [x] if w is None else [x, w], dy, retain_graph=True)
        back, bsize = _turn64(G, cos, sin, "half", 0, -1.0)
        if w is None:
            _near(dx, back, E32 * back.abs() + 4 * E32 * bsize, "dx")
            continue
        g, gs = back * W, bsize * W.abs()
        ref = r * (g - X * r * r * (g * X).mean(-1, keepdim=True))
        _near(dx, ref, E32 * ref.abs() + 64 * E32 * r * (gs + X.abs() * r * r * (gs * X.abs()).mean(-1, keepdim=True)), "dx")
        ref = (back * X * r).sum((0, 1))
        _near(dw[0], ref, E32 * ref.abs() + (64 + T * x.shape[1] / 8) * E32 * (bsize * X.abs() * r).sum((0, 1)), "dw")


def test_scaling_with_entries_of_other_uses():
    """A configuration's dict may hold entries that the frequencies do not depend on, lists among them."""
    from torchllmtuner_b200 import ops
    scaling = {"rope_type": "linear", "factor": 3.0, "mrope_section": [8, 12, 12], "type": "linear"}
    pos = torch.arange(70, device=DEV)
    cos, sin = ops.rope_tables(pos, 64, 1e4, scaling=scaling)
    ang = torch.arange(70, dtype=torch.float64)[:, None] * torch.tensor([1e4 ** (-2 * j / 64) / 3.0 for j in range(32)], dtype=torch.float64)
    bound = (math.pi + 4) * E32 + 2.0 ** -50 * ang
    assert ((cos.cpu().double() - ang.cos()).abs() <= bound).all() and ((sin.cpu().double() - ang.sin()).abs() <= bound).all()
