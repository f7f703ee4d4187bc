"""Rows of logits where parts of rows meet, where rows end, and of what is not a number or not allowed."""
import math

import pytest

from conftest import announce
from sequence_reference import worst
from tokens_reference import TYPES, LogProbs, teacher

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

INF = float("inf")


def _borders(vocab):
    """Both ends of a row and both sides of whatever a part may end at: parts are whole rounds of 256 vectors of 4 or 8
    elements, counted from the first multiple of 16 bytes, which is up to 7 elements from the row's begin."""
    at = set(range(8)) | set(range(vocab - 16, vocab))
    for border in range(1024, vocab, 1024):
        at |= set(range(border - 1, border + 8))
    return torch.tensor(sorted(c for c in at if c < vocab), device="cuda")


# 16 bits: a little beside multiples of 8192, 32 bits: of 4096, where a part has the row's end and nothing else
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [12287, 12289, 20481, 24571, 24577, 32767, 32769, 40963, 49153, 65535, 65537])
def test_entries_at_the_borders(vocab, dtype):
    """A teacher that names the columns at the borders of parts, in rows of every misalignment: each has its term."""
    from gear_amd import ops
    announce("distill at borders %s %d" % (dtype, vocab))
    g = torch.Generator(device="cuda").manual_seed(vocab)
    wide = (torch.randn(9, vocab + 3, generator=g, device="cuda") * 2).to(dtype)
    for x in (wide[:, 1:1 + vocab], wide[:, :vocab].contiguous()):
        ref = LogProbs(x, 1.0)
        for best in _borders(vocab).split(64):
            best = best.expand(9, -1).contiguous()
            t = torch.randn(best.shape, generator=g, device="cuda")
            dloss = 1 + torch.rand(9, generator=g, device="cuda")
            _, lse = ops.distill(x, best, t)
            got = ops.distill_backward(dloss, x, best, t, lse)
            q, q_error, _ = teacher(best, t, vocab)
            weight, error = (torch.zeros_like(ref.p).scatter_(1, best, v) for v in (q, q_error))
            a = dloss.double()[:, None]
            want, bound = ref.gradient(a, torch.zeros_like(a), -a * weight, dtype, ref.lse, a)
            assert worst(got, want, bound + a * (error + 2.0 ** -24 * 66 * weight)) <= 1, (x.is_contiguous(), best[0, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [2049, 12289, 24577, 32767, 32769, 65537])
def test_tokens_at_the_ends(vocab, dtype):
    """The given token's term in the first and last columns, in rows of every misalignment."""
    from gear_amd import ops
    announce("log_probs_backward at the ends %s %d" % (dtype, vocab))
    g = torch.Generator(device="cuda").manual_seed(vocab)
    tokens = torch.cat([torch.arange(8), torch.arange(vocab - 16, vocab)]).cuda().repeat_interleave(8)
    x = (torch.randn(len(tokens), vocab, generator=g, device="cuda") * 2).to(dtype)
    ref = LogProbs(x, 1.0)
    dl = 1 + torch.rand(len(tokens), generator=g, device="cuda")
    outs = ops.token_log_probs(x, tokens)
    got = ops.token_log_probs_backward(dl, None, x, tokens, outs[2], None)
    a = dl.double()[:, None]
    at = torch.zeros_like(ref.p).scatter_(1, tokens[:, None], 1.0)
    want, bound = ref.gradient(-a, torch.zeros_like(a), a * at, dtype, ref.lse, a)
    assert worst(got, want, bound) <= 1


def _all_nan(*tensors):
    return all(bool(torch.isnan(t).all()) for t in tensors)


# rows of lane groups, of a wave, of a workgroup, of one of 1024 threads, of several parts that are joined
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 5, 70, 600, 2000, 3000, 9001, 33025, 70001, 150001])
def test_nothing_but_nan(vocab, dtype):
    """NaN is its row's whatever else the row holds: alone, among tokens that are not allowed, among the lowest numbers.  A
    row that allows nothing and holds no NaN is one that allows nothing, and a row that is passed over is not looked at."""
    from gear_amd import ops
    announce("rows of nothing but NaN %s %d" % (dtype, vocab))
    nan, low = float("nan"), torch.finfo(dtype).min
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(9, vocab, generator=g, device="cuda").to(dtype)
    x[0] = nan
    x[1:4] = -INF
    x[1, 0], x[2, vocab - 1], x[3, vocab // 2] = nan, nan, nan
    x[4] = low
    x[4, vocab // 3] = nan
    x[5] = -INF  # nothing is allowed
    x[6] = nan   # passed over
    tokens = torch.tensor([0, vocab - 1, 0, vocab - 1, 0, 0, -1, 0, vocab - 1], device="cuda")
    first = [0, 0, vocab - 1, vocab // 2, vocab // 3]
    for top in sorted({0, 1, min(5, vocab), min(64, vocab)}):
        logp, entropy, lse, value, best = ops.token_log_probs(x, tokens, top=top)
        assert _all_nan(logp[:5], entropy[:5], lse[:5])
        assert float(logp[5]) == float(lse[5]) == -INF and float(entropy[5]) == 0
        assert float(logp[6]) == float(lse[6]) == float(entropy[6]) == 0
        assert bool(torch.isfinite(torch.stack([logp[7:], lse[7:], entropy[7:]])).all())
        if top:
            assert _all_nan(value[:5]) and best[:5, 0].tolist() == first
            assert bool((value[5:7] == -INF).all()) and bool((best[6] == -1).all()) and best[5].tolist() == list(range(top))
    one = torch.ones(9, device="cuda")
    for a, b in ((one, None), (None, one), (one, one)):
        grad = ops.token_log_probs_backward(a, b, x, tokens, lse, entropy)
        assert _all_nan(grad[:5]) and float(grad[5:7].abs().sum()) == 0 and bool(torch.isfinite(grad[7:]).all())
    best = tokens[:, None].clone()
    t = torch.zeros(9, 1, device="cuda")
    loss, lse = ops.distill(x, best, t)
    assert _all_nan(loss[:5], lse[:5]) and float(loss[5]) == INF and float(lse[5]) == -INF
    assert float(loss[6]) == float(lse[6]) == 0 and bool(torch.isfinite(torch.stack([loss[7:], lse[7:]])).all())
    grad = ops.distill_backward(one, x, best, t, lse)
    assert _all_nan(grad[:5]) and float(grad[5:7].abs().sum()) == 0 and bool(torch.isfinite(grad[7:]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [2, 9, 700, 3000, 70001])
def test_nothing_but_the_lowest(vocab, dtype):
    """Rows of a type's lowest number allow nothing in 32 bits and in bfloat16; in fp16 it is a logit like any other, and all of
    them are as probable as each other."""
    from gear_amd import ops
    announce("rows of the lowest number %s %d" % (dtype, vocab))
    x = torch.full((3, vocab), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    tokens, one = torch.tensor([0, vocab - 1, -1], device="cuda"), torch.ones(3, device="cuda")
    logp, entropy, lse, value, best = ops.token_log_probs(x, tokens, top=2)
    grad = ops.token_log_probs_backward(one, None, x, tokens, lse, None)
    loss, _ = ops.distill(x, tokens[:, None], 0 * one[:, None])
    assert best.tolist() == [[0, 1], [0, 1], [-1, -1]]
    if dtype == torch.float16:
        # S is a sum of equal numbers in 32 bits (200 roundings, LogProbs), its logarithm has a few more; lse is rounded once as -65504 is
        logs = math.log(vocab)
        bound = 2.0 ** -24 * (220 + 8 * logs)
        for got in (-logp[:2], entropy[:2], -value[:2, 0], loss[:2]):
            assert float((got.double() - logs).abs().max()) <= 2 * bound
        assert float((lse[:2].double() + 65504 - logs).abs().max()) <= bound + 2.0 ** -9
        assert float(grad[0, 0]) > 0 and float(grad[0, 1]) < 0
    else:
        assert bool((logp[:2] == -INF).all()) and bool((lse[:2] == -INF).all()) and bool((value[:2] == -INF).all())
        assert float(entropy.abs().sum()) == 0 and float(grad.abs().sum()) == 0 and bool((loss[:2] == INF).all())


@pytest.mark.parametrize("vocab", [6, 900, 9001])
@pytest.mark.parametrize("far", [-3000.0, 500.0, 70000.0])
def test_gradients_far_from_zero(far, vocab):
    """p is exp(z - lse) of the lse that is given: one rounding of a difference near 0, however large both are."""
    from gear_amd import ops
    announce("gradients of far logits %g %d" % (far, vocab))
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(5, vocab, generator=g, device="cuda") + far
    scale = float(torch.tensor(0.7))
    tokens, one = torch.zeros(5, dtype=torch.int64, device="cuda"), torch.ones(5, device="cuda")
    _, entropy, lse, _, _ = ops.token_log_probs(x, tokens, scale=scale)
    d = x.double() * scale - lse.double()[:, None]
    p, h = torch.exp(d.clamp(max=0)), entropy.double()[:, None]  # (above 0 by no more than lse is off)
    # d and log2 e are rounded, their product is, the power and two products are: each a unit of d or of the result
    off = 2.0 ** -24 * (4 * d.abs() + 12)
    token = torch.nn.functional.one_hot(tokens, vocab)
    got = ops.token_log_probs_backward(one, None, x, tokens, lse, entropy, scale=scale)
    assert worst(got, scale * (token - p), scale * (p * off + 2.0 ** -24 * 4 * token)) <= 1
    got = ops.token_log_probs_backward(None, one, x, tokens, lse, entropy, scale=scale)
    slope = d.clamp(max=0) + h
    assert worst(got, -scale * p * slope, scale * p * (off * (slope.abs() + 1) + 2.0 ** -24 * 8 * (d.abs() + h))) <= 1
    t = torch.zeros(5, 1, device="cuda")
    got = ops.distill_backward(one, x, tokens[:, None], t, lse, scale=scale)
    assert worst(got, scale * (p - token), scale * (p * off + 2.0 ** -24 * 4 * token)) <= 1
