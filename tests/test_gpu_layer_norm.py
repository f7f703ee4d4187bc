"""Layer norm of rows, with and without a residual, and its gradients, against 64 bits."""
import pytest

from conftest import announce
from sequence_reference import UNIT, worst
from tokens_reference import TYPES, LayerNorm, rounded

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

WIDTHS = [1, 2, 3, 7, 8, 9, 16, 31, 33, 64, 65, 100, 127, 128, 130, 255, 257, 500, 512, 520, 1000, 1023, 1024, 1025, 2047, 2048, 2056, 4095,
          4097, 5000, 8191, 8193, 8200, 16383, 16384]


def _weights_off(dw, ref, error, dtype):
    return worst(dw, ref, error + rounded(ref, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_forward_and_backward(width, dtype):
    from gear_amd import ops
    for rows, residual, beside in ((1, False, False), (3, True, True), (37, False, True), (1030 if width < 3000 else 130, True, False)):
        g = torch.Generator(device="cuda").manual_seed(width + rows)
        announce("layer_norm %s %d x %d residual=%s beside=%s" % (dtype, rows, width, residual, beside))
        draw = lambda mean=0.0: (torch.randn(rows, 3, width, generator=g, device="cuda") * 2 + mean).to(dtype)  # noqa: E731
        pick = lambda t: t[:, 1] if beside else t[:, 1].contiguous()  # noqa: E731
        x, r, dy, dsum = pick(draw(3.0)), pick(draw()), pick(draw()), pick(draw())
        own = rows % 2 == 1  # weights of the rows' type, or of 32 bits
        w, b = ((t * 0.3 + 1).to(dtype if own else torch.float32) for t in torch.randn(2, width, generator=g, device="cuda"))
        if residual:
            y, u = ops.layer_norm(x, w, b, residual=r, eps=1e-5)
            total = x.double() + r.double()
            assert u.dtype == dtype and worst(u, total, rounded(total, dtype) + (0 if dtype == torch.float32 else 2.0 ** -24) * total.abs()) <= 1
        else:
            y, u = ops.layer_norm(x, w, b, eps=1e-5), x
        ref = LayerNorm(u, w, b, 1e-5, dy, dsum if residual else None)
        assert y.dtype == dtype and y.is_contiguous() and worst(y, ref.y, ref.y_bound) <= 1
        dx, dw, db = ops.layer_norm_backward(dy, u, w, b, dsum=dsum if residual else None, eps=1e-5)
        assert dx.dtype == dtype and dw.dtype == db.dtype == w.dtype
        assert worst(dx, ref.dx, ref.dx_bound) <= 1
        assert _weights_off(dw, ref.dw, ref.dw_error, w.dtype) <= 1 and _weights_off(db, ref.db, ref.db_error, w.dtype) <= 1
        again = ops.layer_norm_backward(dy, u, w, b, dsum=dsum if residual else None, eps=1e-5)
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("dtype", TYPES)
def test_without_weights_and_rows(dtype):
    from gear_amd import ops
    announce("layer_norm without weights %s" % dtype)
    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy = (torch.randn(5, 4, 96, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.rand(96, generator=g, device="cuda")
    ref = LayerNorm(x, None, None, 1e-3, dy)
    assert worst(ops.layer_norm(x, eps=1e-3).view(20, 96), ref.y, ref.y_bound) <= 1
    dx, dw, db = ops.layer_norm_backward(dy, x, eps=1e-3)
    assert dw is None and db is None and worst(dx.view(20, 96), ref.dx, ref.dx_bound) <= 1
    dx, dw, db = ops.layer_norm_backward(dy, x, None, w, eps=1e-3)
    assert dw is None and _weights_off(db, ref.db, ref.db_error, w.dtype) <= 1
    dx, dw, db = ops.layer_norm_backward(dy, x, w, eps=1e-3)
    assert db is None and _weights_off(dw, ref.dw, ref.dw_error, w.dtype) <= 1
    # no rows: no sums
    none = x[:0]
    assert ops.layer_norm(none, w).shape == (0, 4, 96)
    dx, dw, db = ops.layer_norm_backward(none, none, w, w)
    assert dx.shape == (0, 4, 96) and float(dw.abs().sum() + db.abs().sum()) == 0
    one = ops.layer_norm(x[0, 0], w, w)  # a row by itself
    assert torch.equal(one, ops.layer_norm(x, w, w)[0, 0])


def test_far_from_zero_and_not_finite():
    """A small deviation around a large mean keeps its digits; a row that holds NaN or infinity is its own affair."""
    from gear_amd import ops
    announce("layer_norm far from zero")
    g = torch.Generator(device="cuda").manual_seed(2)
    x = 1000 + torch.randn(64, 1024, generator=g, device="cuda")
    ref = LayerNorm(x, None, None, 1e-5, x)
    # the mean is off by up to 26 roundings of 1000, n by as much over a deviation of 1
    assert float((ops.layer_norm(x).double() - ref.y).abs().max()) < 64 * 2.0 ** -24 * 1000
    clean = ops.layer_norm(x)
    x[5, 7], x[9, 1000] = float("nan"), float("inf")
    got = ops.layer_norm(x)
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[[5, 9]] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], clean[~bad])
    flat = torch.full((3, 100), 2.5, device="cuda")  # no deviation: the bias
    assert float(ops.layer_norm(flat).abs().max()) == 0


def test_gradients_against_differences():
    from gear_amd import sequence
    announce("layer_norm: gradients against differences")
    g = torch.Generator(device="cuda").manual_seed(4)
    x, r, gy, gs = torch.randn(4, 3, 10, generator=g, device="cuda")
    w, b = torch.randn(2, 10, generator=g, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, r, w, b)]
    y, u = sequence.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1], eps=0.1)
    ((y * gy).sum() + (u * gs).sum()).backward()
    assert torch.equal(leaves[0].grad, leaves[1].grad)

    def f(x, r, w, b):
        u = x + r
        c = u - u.mean(-1, keepdim=True)
        return ((c / torch.sqrt(c.square().mean(-1, keepdim=True) + 0.1) * w + b) * gy.double() + u * gs.double()).sum()

    h = 1e-5
    for k, leaf in enumerate(leaves):
        for i in range(leaf.numel()):
            at = [t.detach().double() for t in leaves]
            step = torch.zeros(leaf.numel(), dtype=torch.float64, device="cuda")
            step[i] = h
            up, down = list(at), list(at)
            up[k], down[k] = at[k] + step.view(leaf.shape), at[k] - step.view(leaf.shape)
            # differences: h^2 times a third derivative of O(100); 32-bit gradients of O(10)
            assert abs(float((f(*up) - f(*down)) / (2 * h)) - float(leaf.grad.flatten()[i])) < 2e-5
