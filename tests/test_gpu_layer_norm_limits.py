"""LayerNorm at the limits of its rows and values, against the formula in 64 bits under the bounds of test_gpu_block_ops.py."""
import pytest
import torch
from test_gpu_block_ops import TYPES, _norm_check, _rand

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
