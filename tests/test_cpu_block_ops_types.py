"""Rotations of operands wider than 32 bits, without a GPU."""
import pytest
import torch

from torchllmtuner_b200 import ops


@pytest.mark.parametrize("tables", [torch.float32, torch.float64])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotation_of_fp64_operands_stays_in_64_bits(layout, tables):
    """The operand's type is the rotation's: products and the one sum of a channel are each off by half a step of fp64, four of them in all."""
    T, H, d, P, off = 9, 3, 20, 6, 4
    g = torch.Generator().manual_seed(0)
    ang = torch.rand(T, P, generator=g, dtype=torch.float64) * 6
    cos, sin = ang.cos().to(tables), ang.sin().to(tables)
    x = torch.randn(T, H, d, generator=g, dtype=torch.float64)
    first = torch.arange(P) + off if layout == "half" else 2 * torch.arange(P) + off
    second = first + (P if layout == "half" else 1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    for inverse in (False, True):
        t = -s if inverse else s
        want = x.clone()
        want[..., first], want[..., second] = x[..., first] * c - x[..., second] * t, x[..., second] * c + x[..., first] * t
        got = ops.rope(x, cos, sin, layout=layout, offset=off, inverse=inverse)
        assert got.dtype == torch.float64 and (got - want).abs().max() <= 4 * 2.0 ** -53 * 2 * x.abs().max()
    want = ops.rope(x, cos, sin, layout=layout, offset=off)
    for y in ops.qk_norm_rope(x, x, None, None, cos, sin, 0.0, layout=layout, offset=off, norm=False):
        assert torch.equal(y, want)
    # the norm is that of rms_norm (fp32), the rotation behind it the operand's
    w = torch.randn(d, generator=g, dtype=torch.float64)
    for y in ops.qk_norm_rope(x, x, w, w, cos, sin, 1e-6, layout=layout, offset=off, norm=True):
        assert torch.equal(y, ops.rope(ops.rms_norm(x, w, 1e-6), cos, sin, layout=layout, offset=off))


def test_rotation_of_fp64_operands_has_exact_gradients():
    ang = torch.rand(3, 2, dtype=torch.float64)
    for layout in ("half", "interleaved"):
        x = torch.randn(3, 2, 6, dtype=torch.float64, requires_grad=True)
        assert torch.autograd.gradcheck(lambda t: ops.rope(t, ang.cos(), ang.sin(), layout=layout, offset=1), (x,))  # noqa: B023
