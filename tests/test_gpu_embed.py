"""Rows of a table by token, and the table's gradient, against 64 bits."""
import pytest

from conftest import announce
from sequence_reference import worst
from tokens_reference import TYPES, embed, embed_backward

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _tokens(kind, n, vocab, g):
    draw = lambda lo, hi: torch.randint(lo, hi, (n,), generator=g, device="cuda")  # noqa: E731
    if kind == "any":
        return draw(-2, vocab + 2)  # some are none
    if kind == "one":
        return torch.full((n,), vocab - 1, device="cuda")
    if kind == "none":
        return torch.full((n,), -1, device="cuda")
    if kind == "apart":
        return torch.randperm(max(n, vocab), generator=g, device="cuda")[:n]
    if kind == "hot":  # most rows go to one token, in a table with long gaps
        return torch.where(draw(0, 10) < 7, vocab // 3, draw(0, vocab))
    return torch.sort(draw(0, vocab)).values


CASES = [  # n, vocab, width, kind
    (0, 7, 5, "any"), (1, 1, 1, "any"), (1, 3, 8, "any"), (5, 2, 3, "any"), (63, 10, 17, "any"), (300, 40, 130, "any"),
    (128, 1025, 256, "any"), (1000, 9, 7, "one"), (1000, 9, 64, "none"), (777, 5000, 40, "apart"), (4096, 300, 512, "any"),
    (4097, 300, 513, "sorted"), (9000, 70000, 24, "hot"), (33000, 1000, 96, "hot"), (40000, 2, 8, "any"), (2500, 3, 2049, "any"),
    (150000, 65536, 16, "any"), (300001, 257, 33, "hot"), (200, 12, 5000, "hot")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,width,kind", CASES)
def test_forward_and_gradient(n, vocab, width, kind, dtype):
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(n + width)
    announce("embed %s n=%d vocab=%d width=%d %s" % (dtype, n, vocab, width, kind))
    tokens = _tokens(kind, n, vocab, g)
    tokens = tokens.int() if width % 2 else tokens
    # tables and gradients that are slices of wider ones, at odd addresses
    table = torch.randn(vocab, width + 3, generator=g, device="cuda").to(dtype)[:, 1:width + 1]
    dout = torch.randn(n, 2, width, generator=g, device="cuda").to(dtype)[:, 1]
    if kind == "any" and n > 2:
        dout = dout.clone()
        dout[(tokens < 0) | (tokens >= vocab)] = float("nan")  # what belongs to no token is not looked at
    out = ops.embed_tokens(tokens, table, scale=3.0)
    grad = ops.embed_tokens_backward(dout, tokens, vocab, scale=0.3)
    assert out.shape == (n, width) and grad.shape == (vocab, width) and out.dtype == grad.dtype == dtype
    ref, bound = embed(tokens, table, 3.0)
    assert worst(out, ref, bound) <= 1
    ref, bound = embed_backward(dout, tokens, vocab, float(torch.tensor(0.3)))
    assert worst(grad, ref, bound) <= 1
    assert torch.equal(grad, ops.embed_tokens_backward(dout, tokens, vocab, scale=0.3))  # the same bits


def test_shapes():
    from gear_amd import ops
    announce("embed: shapes")
    table = torch.arange(12.0, device="cuda").view(4, 3)
    tokens = torch.tensor([[[0, 3], [-1, 4]]], device="cuda")
    out = ops.embed_tokens(tokens, table)
    assert out.tolist() == [[[[0.0, 1.0, 2.0], [9.0, 10.0, 11.0]], [[0.0] * 3, [0.0] * 3]]]
    assert ops.embed_tokens(tokens[0, 0, 1], table, scale=2.0).tolist() == [18.0, 20.0, 22.0]
    assert ops.embed_tokens(torch.zeros(2, 0, dtype=torch.int32, device="cuda"), table).shape == (2, 0, 3)
    assert ops.embed_tokens(tokens, table[:0]).abs().sum() == 0  # no table: no tokens
    assert ops.embed_tokens_backward(out, tokens, 0).shape == (0, 3)
    grad = ops.embed_tokens_backward(torch.ones(1, 2, 2, 3, device="cuda"), tokens, 5)
    assert grad.sum(1).tolist() == [3.0, 0.0, 0.0, 3.0, 3.0]
    # one row for all tokens, a row of one element for all columns
    row = torch.ones(1, 3, device="cuda").expand(4, 3)
    assert torch.equal(ops.embed_tokens_backward(row, tokens.flatten(), 5), grad)


def test_gradient_against_differences():
    """(f(t + h) - f(t - h)) / 2 h of a linear function in 64 bits: exact but for the roundings."""
    from gear_amd import sequence
    announce("embed: gradient against differences")
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(5, 6, generator=g, device="cuda").requires_grad_()
    tokens = torch.tensor([4, 0, 4, 4, -1, 2], device="cuda")
    weight = torch.randn(6, 6, generator=g, device="cuda")
    (sequence.embed_tokens(tokens, table, scale=1.5) * weight).sum().backward()
    f = lambda t: (1.5 * t[tokens.clamp(min=0)] * (tokens >= 0)[:, None] * weight.double()).sum()  # noqa: E731
    for i in range(5):
        for j in range(6):
            step = torch.zeros(5, 6, dtype=torch.float64, device="cuda")
            step[i, j] = 0.5
            assert abs(float(f(table.detach().double() + step) - f(table.detach().double() - step) - table.grad[i, j])) < 1e-5
