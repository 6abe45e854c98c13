"""Linear layers whose products take each of the kernels' cuts, gradients into an owner's buffer at any width, special values one row each: against the
formulas in 64 bits of test_gpu_block_ops.py and under its bounds."""
import pytest
import torch
from test_gpu_block_ops import DEV, E32, TYPES, _act64, _linear_check, _linear_run, _near, _rand, _u

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- how the products are cut
def _pitch(n):
    """Elements between the rows of a buffer of n columns: on 128 bytes where that adds at most an eighth, else on 16."""
    lines = (n + 63) // 64 * 64
    return lines if lines - n <= n // 8 else (n + 7) // 8 * 8


def _kind(rows, columns, depth, lda, ldb, gradient, act=0, res=False, pre=False):
    """(CTAs of a tile, more than 256 columns, cut along the depth, how the last column of tiles is) of the product's cut."""
    from torchllmtuner_b200.ops.cuda_ext import load
    ctas, bn, parts = load().linear_cut(rows, columns, depth, lda, ldb, gradient, act, res, pre)
    rest = columns % bn
    last = "whole" if rest == 0 else "only" if columns < bn else "narrow" if rest <= 256 else "narrow, second product"
    return ctas, bn > 256, parts > 1, last


CODES = {None: 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "relu": 4}


def _check_cuts(M, K, N, act, res, y=None, dx=None, dw=None):
    """A change of the estimate must not empty these tests: the cut that a case is there for is asserted."""
    lddz = _pitch(N) if act else N
    if y is not None:
        assert _kind(M, N, K, K, K, False, CODES[act], res, act is not None) == y
    if dx is not None:
        assert _kind(M, K, N, lddz, K, True) == dx
    if dw is not None:
        assert _kind(N, K, M, lddz, K, True) == dw


PATHS = [
    # parts along K joined by the second launch: one CTA and pairs, whole and narrow last tiles, one row
    (130, 4608, 200, None, False, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, None, True, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "gelu", False, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "gelu", True, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "gelu_tanh", False, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "gelu_tanh", True, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "silu", False, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "silu", True, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "relu", False, dict(y=(1, False, True, "narrow"))),
    (130, 4608, 200, "relu", True, dict(y=(1, False, True, "narrow"))),
    (200, 2304, 1024, "gelu", True, dict(y=(1, False, True, "whole"))),
    (200, 2304, 1024, "gelu_tanh", False, dict(y=(1, False, True, "whole"))),
    (144, 5488, 136, "gelu", False, dict(y=(2, False, True, "narrow"))),
    (232, 4504, 200, None, False, dict(y=(2, False, True, "narrow"))),
    (1, 3032, 64, None, True, dict(y=(1, False, True, "whole"))),
    # more than 256 columns: a second product per slice, one accumulator
    (4368, 240, 1168, None, False, dict(y=(2, True, False, "narrow"))),
    (1464, 8, 3168, "silu", True, dict(y=(2, True, False, "whole"))),
    (5784, 8, 912, "silu", False, dict(y=(2, True, False, "narrow, second product"))),
    (14768, 624, 368, None, False, dict(y=(2, True, False, "only"))),
    (2464, 7328, 608, "relu", False, dict(y=(2, True, True, "narrow, second product"))),
    (304, 6088, 3216, None, False, dict(y=(2, True, True, "narrow"))),
    (1112, 7712, 1056, "relu", True, dict(y=(2, True, True, "whole"))),
    # the same of the gradients' products
    (16384, 1152, 4608, "gelu_tanh", False, dict(dx=(2, True, False, "whole"), dw=(2, True, False, "whole"))),
    (944, 5040, 152, None, False, dict(dx=(2, True, False, "narrow"))),
    (8128, 568, 144, "gelu", False, dict(dx=(2, True, False, "narrow, second product"))),
    (17992, 312, 168, None, False, dict(dx=(2, True, False, "only"))),
    (5984, 4704, 152, None, False, dict(dw=(2, True, True, "narrow"))),
    (9856, 1808, 264, None, True, dict(dw=(2, True, True, "narrow, second product"))),
    (8056, 288, 2536, "relu", False, dict(dw=(2, True, True, "whole"))),
    (3656, 152, 152, None, False, dict(dw=(2, False, True, "narrow"))),
]


@pytest.mark.parametrize("M,K,N,act,res,cuts", PATHS, ids=lambda v: "-".join(sorted(v)) if isinstance(v, dict) else str(v))
def test_linear_act_cuts(M, K, N, act, res, cuts):
    _check_cuts(M, K, N, act, res, **cuts)
    x, w = _rand(M, K, seed=1).requires_grad_(), _rand(N, K, seed=2, std=K ** -0.5).requires_grad_()
    b, dy = _rand(N, seed=3, std=0.5).requires_grad_(), _rand(M, N, seed=5)
    r = _rand(M, N, seed=4).requires_grad_() if res else None
    outs = _linear_run(x, w, b, r, act, dy)
    _linear_check(x.detach(), w.detach(), b.detach(), r.detach() if res else None, act, dy, outs)


# -------------------------------------------------------------------------------------------- gradients with an owner
class _Queue:
    """A collective queue that never gives a product a slice to carry."""

    def __bool__(self):
        return True

    def take(self, flops):
        return None, ()


@pytest.mark.parametrize("queue", [False, True], ids=["", "queue"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("M,K,N,columns_first", [(300, 201, 137, False), (300, 201, 136, False), (65, 40, 72, True), (130, 33, 7, True), (1, 8, 8, False)])
def test_owners_buffer_at_any_width(M, K, N, columns_first, act, dtype, queue):
    """Widths that are no multiple of 8 and weights stored columns first: the weight's gradient is written to `main_grad` by the first micro-batch and
    added to by the second; x and bias get what they get without an owner."""
    from torchllmtuner_b200 import ops
    from torchllmtuner_b200.parallel import symm
    x, b = _rand(M, K, seed=1).requires_grad_(), _rand(N, seed=3).requires_grad_()
    w = _rand(K, N, seed=2, std=K ** -0.5).t() if columns_first else _rand(N, K, seed=2, std=K ** -0.5)
    w = w.detach().requires_grad_()
    dys = [_rand(M, N, seed=4), _rand(M, N, seed=5)]
    plain = [_linear_run(x, w, b, None, act, dy) for dy in dys]
    w.main_grad, w.main_grad_initialized = torch.full((N, K), 7.0, device=DEV, dtype=TYPES[dtype]), False
    um, total, bound = _u(TYPES[dtype]), 0.0, 0.0
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    size = x.detach().double().abs() @ w.detach().double().abs().t() + b.detach().double().abs()
    _, slope, curve = _act64(z, act)
    for i, dy in enumerate(dys):
        y = ops.linear_act(x, w, b, activation=act)
        symm.set_active_queue(_Queue() if queue else None)
        try:
            dx, dw, db = torch.autograd.grad(y, (x, w, b), dy, allow_unused=True)
        finally:
            symm.set_active_queue(None)
        assert dw is None and w.main_grad_initialized
        assert torch.equal(db, plain[i]["db"])
        # the products add in fp32 in another order: half a step of bf16 on either side of the same sum
        assert ((dx.double() - plain[i]["dx"].double()).abs() <= 2.02 * _u(torch.bfloat16) * plain[i]["dx"].double().abs() + 2 * (N + 8) * E32 * (
            (1.2 * dy.double().abs()) @ w.detach().double().abs())).all()
        dz = dy.double() * slope
        edz = _u(torch.bfloat16) * dz.abs() + dy.double().abs() * (curve * (_u(torch.bfloat16) * z.abs() + (K + 8) * E32 * size) + 16 * E32 * (1 + z.abs())) if act else torch.zeros_like(dz)
        total = total + dz.t() @ x.detach().double()
        # each product's error, and a rounding of the buffer each time
        bound = bound + edz.t() @ x.detach().double().abs() + (M + 8) * E32 * ((dz.abs() + edz).t() @ x.detach().double().abs())
        bound = bound + um * (total.abs() + bound) + 1e-30
        _near(w.main_grad, total, bound, f"main_grad after {i + 1}")


# --------------------------------------------------------------------------------------------------- special values
def test_special_values_in_rows_of_their_own():
    """NaN, infinities and the largest values, one to a row and each multiplied by one alone: what the formula gives, NaN where it gives NaN."""
    from torchllmtuner_b200 import ops
    z = torch.tensor([float("nan"), float("inf"), float("-inf"), 3e38, -3e38, 1e30, -1e30, 1e4, -1e4, 40.0, -40.0, 11.0, -11.0, -8.0, -3.0, -0.7, 0.0, 0.7, 3.0, 8.0], device=DEV)
    x = z.bfloat16()[:, None].requires_grad_()
    w = torch.ones(9, 1, device=DEV, dtype=torch.bfloat16)
    for act in (None, "relu", "gelu", "gelu_tanh", "silu"):
        y = ops.linear_act(x, w, activation=act)
        ref, slope, _ = _act64(x.detach().double(), act)
        ref = ref.expand(-1, 9)
        assert torch.equal(y.isnan(), ref.isnan()), (act, y, ref)
        assert torch.equal(y.isinf(), ref.isinf()) and (y[y.isinf()].double() == ref[y.isinf()]).all(), (act, y, ref)
        fin = ref.isfinite()
        # a rounding to bf16, and 16 steps of fp32 of z for the function
        assert ((y.double() - ref).abs()[fin] <= (_u(torch.bfloat16) * ref.abs() + 16 * E32 * x.detach().double().abs())[fin]).all(), (act, y, ref)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert dx[0].isnan().all() or act in (None, "relu")            # NaN has no slope; without one, and at relu's, the gradient passes
        rows = x.detach()[:, 0].isfinite()
        want = (9 * slope)[rows]
        # dz is rounded to bf16, and so is the sum of nine
        assert ((dx.detach()[rows].double() - want).abs() <= 2.02 * _u(torch.bfloat16) * want.abs() + 9 * 16 * E32 * (1 + x.detach()[rows].double().abs().clamp(max=100))).all(), (act, dx, slope)


# ------------------------------------------------------------------------------------------------ sizes at the limits
def test_linear_act_refuses_sizes_past_its_range():
    """Rows and features count up to 2^31 - 512 (a tile's end is still a 32-bit number): more is refused before anything is allocated or launched."""
    from torchllmtuner_b200 import ops
    most = (1 << 31) - 512
    row, w = torch.zeros(1, 8, device=DEV, dtype=torch.bfloat16), torch.zeros(8, 8, device=DEV, dtype=torch.bfloat16)
    before = torch.cuda.memory_allocated()
    for rows in (most + 1, (1 << 31) - 1, 1 << 31, (1 << 32) + 5):
        with pytest.raises(RuntimeError, match="rows"):
            ops.linear_act(row.expand(rows, 8), w)
        with pytest.raises(RuntimeError, match="features"):
            ops.linear_act(row, row.expand(rows, 8))
        with pytest.raises(RuntimeError, match="features"):
            ops.linear_act(row[:, :1].expand(1, rows), row[:, :1].expand(8, rows))
    assert torch.cuda.memory_allocated() == before


def test_linear_act_of_the_most_rows():
    """2^31 - 512 rows of one feature: every value of y and dx is a product by two, exact."""
    from torchllmtuner_b200 import ops
    x = torch.empty((1 << 31) - 512, 1, device=DEV, dtype=torch.bfloat16).normal_().requires_grad_()
    w = torch.full((1, 1), 2.0, device=DEV, dtype=torch.bfloat16)
    y = ops.linear_act(x, w)
    with torch.no_grad():
        assert torch.equal(y, x * 2)
        dy = torch.empty_like(y).normal_()
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx, dy * 2)
    del x, y, dx, dy
    torch.cuda.empty_cache()


def test_linear_act_one_row_whose_gradient_has_no_row_stride():
    """A single row of the upstream gradient may carry any stride between rows, zero among them."""
    from torchllmtuner_b200 import ops
    x, w, b = _rand(1, 200, seed=1).requires_grad_(), _rand(136, 200, seed=2, std=0.07).requires_grad_(), _rand(136, seed=3).requires_grad_()
    dy = _rand(136, seed=4)
    want = torch.autograd.grad(ops.linear_act(x, w, b), (x, w, b), dy[None])
    for stride in (0, 1, 8, 72):
        got = torch.autograd.grad(ops.linear_act(x, w, b), (x, w, b), dy.as_strided((1, 136), (stride, 1)))
        assert all(torch.equal(p, q) for p, q in zip(got, want)), stride
