"""The pieces of a block under activation checkpointing, in inference mode and after a change of what they saved."""
import pytest
import torch
from test_gpu_block_ops import DEV, _rand

pytestmark = pytest.mark.gpu


def _step(x, w, b, lw, lb, qw, cos, sin):
    from torchllmtuner_b200 import ops
    h = ops.layer_norm(ops.linear_act(x, w, b, activation="gelu", residual=x[:, :1]), lw, lb, 1e-5).view(len(x), 4, 33)
    q, k = ops.qk_norm_rope(h[:, :3], h[:, 3:], qw, None, cos, sin, 1e-6, offset=5, norm=True)
    return torch.cat((q, ops.rope(k, cos, sin, layout="interleaved", offset=1)), 1).flatten(1)


def _step_args():
    ang = torch.rand(90, 10, device=DEV) * 6
    x, w, b = _rand(90, 67, seed=1), _rand(132, 67, seed=2, std=0.1), _rand(132, seed=3)
    return [x, w, b, *(_rand(n, seed=i) for i, n in ((4, 132), (5, 132), (6, 33)))], (ang.cos(), ang.sin())


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_in_the_backward(reentrant):
    """Under activation checkpointing the same bits as without."""
    from torch.utils.checkpoint import checkpoint
    args, tables = _step_args()
    got = []
    for wrap in (lambda *a: _step(*a, *tables), lambda *a: checkpoint(lambda *t: _step(*t, *tables), *a, use_reentrant=reentrant)):
        leaves = [t.clone().requires_grad_() for t in args]
        y = wrap(*leaves)
        y.backward(torch.ones_like(y))
        got.append([y.detach(), *(t.grad for t in leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_inference_mode_gives_the_same_bits():
    args, tables = _step_args()
    want = _step(*args, *tables)
    with torch.inference_mode():
        assert torch.equal(_step(*args, *tables), want)


@pytest.mark.parametrize("index", range(6))
def test_a_saved_tensor_changed_in_place_is_noticed(index):
    args, tables = _step_args()
    leaves = [t.clone().requires_grad_() for t in args]
    mid = [t * 1 for t in leaves]
    y = _step(*mid, *tables)
    with torch.no_grad():
        mid[index].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))
