"""Log probabilities of tokens, entropies, the best tokens, distillation, and the gradients of the logits, against 64 bits."""
import math

import pytest

from conftest import announce
from sequence_reference import worst
from tokens_reference import TYPES, LogProbs, order, teacher

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

INF = float("inf")
# rows of a lane group, of a wave, of a workgroup, of several: with every type's borders, and one to either side
SIZES = [(1, 1), (5, 2), (70, 3), (300, 7), (1, 8), (33, 9), (300, 18), (64, 33), (3, 64), (50, 127), (20, 129), (9, 255), (7, 513),
         (2, 1000), (5, 1024), (4, 1025), (3, 2047), (2, 2048), (3, 2049), (1100, 2500), (2, 4096), (3, 4097), (1, 8193), (1030, 9001),
         (1, 20480), (2, 20481), (1, 33025), (2, 40961), (1025, 41000), (2, 65537), (1, 131073)]


def _logits(rows, vocab, dtype, g, kind, beside):
    x = torch.randn(rows, 2, vocab + 1, generator=g, device="cuda") * 3
    if kind == "far":
        x = x + 500
    x = x.to(dtype)[:, 1, 1:] if beside else x[:, 1, :vocab].to(dtype).contiguous()
    if kind == "masked":
        hidden = torch.rand(rows, vocab, generator=g, device="cuda") < 0.4
        x = x.masked_fill(hidden, -INF)
        x[::7] = -INF  # nothing is allowed there
    if kind == "lowest":
        x = x.masked_fill(torch.rand(rows, vocab, generator=g, device="cuda") < 0.5, torch.finfo(dtype).min)
    if kind == "equal":
        x = torch.full_like(x, 0.25)
    return x


def _check_forward(x, tokens, scale, top, outs):
    rows, vocab = x.shape
    ref = LogProbs(x, scale)
    logp, entropy, lse, value, best = outs
    alive = torch.ones(rows, dtype=torch.bool, device="cuda")
    if tokens is not None:
        alive = (tokens >= 0) & (tokens < vocab)
        at = tokens.clamp(0, vocab - 1).long()[:, None]
        want, d = ref.logp.gather(1, at)[:, 0], ref.d.gather(1, at)[:, 0]
        want = torch.where(ref.none | (x.gather(1, at)[:, 0] == -INF), -INF, want)
        assert worst(logp[alive], want[alive], ref.logp_bound(want, d)[alive]) <= 1
        assert float(logp[~alive].abs().sum() + entropy[~alive].abs().sum() + lse[~alive].abs().sum()) == 0
    else:
        assert logp is None
    assert worst(lse[alive], torch.where(ref.none, -INF, ref.lse)[alive], ref.lse_bound[alive]) <= 1
    assert worst(entropy[alive], torch.where(ref.none, 0.0, ref.entropy)[alive], ref.entropy_bound[alive] + 1e-12) <= 1
    if top:
        want = order(x, top)
        assert best.dtype == torch.int64 and torch.equal(best[alive], want[alive])
        logs = torch.where(ref.none[:, None] | (x.gather(1, want) == -INF), -INF, ref.logp.gather(1, want))
        bound = (ref.s_error[:, None] + 2.0 ** -24 * (4 * ref.d.gather(1, want).abs() + 2 * logs.abs() + 4))
        assert worst(value[alive], logs[alive], bound[alive]) <= 1
        assert bool((best[~alive] == -1).all()) and bool((value[~alive] == -INF).all())
    else:
        assert value is None and best is None
    return ref, alive


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_log_probs(rows, vocab, dtype):
    from gear_amd import ops
    kinds = ["plain", "masked", "far", "lowest", "equal"]
    for turn, kind in enumerate(kinds if rows * vocab < 3000000 else kinds[:2]):
        g = torch.Generator(device="cuda").manual_seed(rows + vocab + turn)
        x = _logits(rows, vocab, dtype, g, kind, beside=turn % 2 == 1)
        scale = (1.0, 0.7)[turn % 2]
        scale = float(torch.tensor(scale))
        tokens = torch.randint(-1, vocab + (rows > 10), (rows,), generator=g, device="cuda")
        tokens = tokens.int() if turn % 2 else tokens
        top = min(vocab, (0, 1, 5, 64, 33)[(turn + rows) % 5])
        announce("log_probs %s %d x %d %s top=%d" % (dtype, rows, vocab, kind, top))
        outs = ops.token_log_probs(x, tokens, scale=scale, top=top)
        ref, alive = _check_forward(x, tokens, scale, top, outs)
        _check_forward(x, None, scale, min(vocab, 64), ops.token_log_probs(x, scale=scale, top=min(vocab, 64)))
        # gradients
        dl, de = torch.randn(2, rows, generator=g, device="cuda")
        live = (alive & ~ref.none)[:, None]
        at = torch.zeros_like(ref.p).scatter_(1, tokens.clamp(0, vocab - 1).long()[:, None], 1.0)
        for a, b in ((dl, de), (dl, None), (None, de)):
            got = ops.token_log_probs_backward(a, b, x, tokens, outs[2], outs[1], scale=scale)
            assert got.dtype == dtype and got.is_contiguous()
            a, b = (torch.zeros(rows, 1, dtype=torch.float64, device="cuda") if t is None else t.double()[:, None] for t in (a, b))
            h = ref.entropy[:, None]
            extra = a.abs() + b.abs() * (1 + h + ref.entropy_bound[:, None] * 2 ** 20)  # (the entropy it is given is off, too)
            want, bound = ref.gradient(-a - b * h, -b, a * at, dtype, ref.lse, extra)
            assert worst(got, torch.where(live, want, 0.0), torch.where(live, bound, 1e-300)) <= 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_distill(rows, vocab, dtype):
    from gear_amd import ops
    for turn, kind in enumerate(("plain", "far", "plain") if rows * vocab < 3000000 else ("plain",)):
        g = torch.Generator(device="cuda").manual_seed(rows + 2 * vocab + turn)
        x = _logits(rows, vocab, dtype, g, kind, beside=turn % 2 == 1)
        count = (min(vocab, 8), 1, 64)[turn]
        announce("distill %s %d x %d %s count=%d" % (dtype, rows, vocab, kind, count))
        scale = (1.0, 0.5, 2.0)[turn]
        if count == 64:  # some named twice, some none, some beyond the vocabulary
            best = torch.randint(-1, vocab + 1, (rows, count), generator=g, device="cuda").int()
        else:
            best = torch.topk(torch.rand(rows, vocab, generator=g, device="cuda"), count).indices
        t = torch.randn(rows, count, generator=g, device="cuda") * 3
        t[torch.rand(rows, count, generator=g, device="cuda") < 0.1] = -INF
        if rows > 3:
            best[2] = -1
            x[2] = float("nan")  # a row that is passed over is not looked at
        loss, lse = ops.distill(x, best, t, scale=scale)
        q, q_error, some = teacher(best, t, vocab)
        ref = LogProbs(torch.where(some[:, None], x, torch.zeros_like(x)), scale)
        at = best.clamp(0, vocab - 1).long()
        logp, d = ref.logp.gather(1, at), ref.d.gather(1, at)
        want = (torch.special.xlogy(q, q) - q * logp).sum(-1)
        each = torch.where(q > 0, torch.log(torch.where(q > 0, q, 1.0)) - logp, 0.0).abs()
        bound = (q_error * (each + 1) + q * (ref.s_error[:, None] + 2.0 ** -24 * (4 * d.abs() + 80 * each + 80))).sum(-1)
        assert worst(loss, torch.where(some, want, 0.0), torch.where(some, bound, 1e-300)) <= 1
        assert worst(lse, torch.where(some, ref.lse, 0.0), torch.where(some, ref.lse_bound, 1e-300)) <= 1
        dloss = torch.randn(rows, generator=g, device="cuda")
        got = ops.distill_backward(dloss, x, best, t, lse, scale=scale)
        weight, error = (torch.zeros_like(ref.p).scatter_add_(1, at, v) for v in (q, q_error))
        a = dloss.double()[:, None]
        want, bound = ref.gradient(a, torch.zeros_like(a), -a * weight, dtype, ref.lse, a.abs())
        bound = bound + scale * a.abs() * (error + 2.0 ** -24 * 66 * weight)  # (weights of one token are added)
        assert worst(got, torch.where(some[:, None], want, 0.0), torch.where(some[:, None], bound, 1e-300)) <= 1


@pytest.mark.parametrize("vocab", [5, 300, 2000, 3000, 50000])
@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite(vocab, dtype):
    """NaN and infinity make their row NaN and no other, gradients with it; they come before all in the order, the lower
    index first."""
    from gear_amd import ops
    announce("log_probs not finite %s %d" % (dtype, vocab))
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(6, vocab, generator=g, device="cuda").to(dtype)
    clean = ops.token_log_probs(x, top=3)
    x[1, vocab - 1], x[3, 2], x[3, 4] = float("nan"), INF, INF
    x[4, 0] = float("nan")
    tokens = torch.zeros(6, dtype=torch.int64, device="cuda")
    logp, entropy, lse, value, best = ops.token_log_probs(x, tokens, top=3)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    for t in (logp, entropy, lse):
        assert bool(torch.isnan(t[bad]).all()) and bool(torch.isfinite(t[~bad]).all())
    for a, b in zip(clean[1:], (entropy, lse, value, best)):
        assert torch.equal(a[~bad], b[~bad])
    assert int(best[1, 0]) == vocab - 1 and best[3, :2].tolist() == [2, 4] and int(best[4, 0]) == 0
    assert best[1, 1:].tolist() == order(x[1:2, :vocab - 1], 2)[0].tolist()
    grad = ops.token_log_probs_backward(torch.ones(6, device="cuda"), torch.ones(6, device="cuda"), x, tokens, lse, entropy)
    assert bool(torch.isnan(grad[bad]).all()) and bool(torch.isfinite(grad[~bad]).all())
    loss, lse = ops.distill(x, tokens[:, None], torch.zeros(6, 1, device="cuda"))
    assert bool(torch.isnan(loss[bad]).all()) and bool(torch.isfinite(loss[~bad]).all())
    grad = ops.distill_backward(torch.ones(6, device="cuda"), x, tokens[:, None], torch.zeros(6, 1, device="cuda"), lse)
    assert bool(torch.isnan(grad[bad]).all()) and bool(torch.isfinite(grad[~bad]).all())
    # a teacher that is not finite is its row's affair too
    t = torch.zeros(6, 1, device="cuda")
    t[0], t[2] = float("nan"), -INF
    loss, lse = ops.distill(x, tokens[:, None], t)
    assert math.isnan(float(loss[0])) and float(loss[2]) == 0 and math.isfinite(float(loss[5]))


@pytest.mark.parametrize("vocab", [40, 700, 3000, 9000, 70000])
def test_ties_and_signs(vocab):
    """Many equal logits, zeros of both signs, a few larger ones among them: the lower index first."""
    from gear_amd import ops
    announce("ties %d" % vocab)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    for rows in (2, 1100):
        x = torch.randint(-2, 3, (rows, vocab), generator=g, device="cuda").float()
        x[0] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.5, -0.0, 0.0)
        x[1, vocab // 2:] = 7.0
        for dtype in TYPES:
            best = ops.token_log_probs(x.to(dtype), top=min(64, vocab))[4]
            assert torch.equal(best, order(x, min(64, vocab)))
            assert torch.equal(ops.token_log_probs(x.to(dtype), top=1)[4], best[:, :1])


@pytest.mark.parametrize("vocab", [5, 20, 64, 130, 513, 2000, 2560, 9000, 33025, 70000])
def test_best_of_few_allowed(vocab):
    """Fewer allowed tokens than are asked for, in few places, and none in a part of every vector's columns; NaN and infinity
    among them: as sorted, the tokens that are not allowed last."""
    from gear_amd import ops
    announce("best of few %d" % vocab)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    at = torch.arange(vocab, device="cuda")
    for rows in (3, 270):
        x = torch.randn(rows, vocab, generator=g, device="cuda")
        few = torch.rand(rows, vocab, generator=g, device="cuda") < 20 / vocab
        for dtype in TYPES:
            per = 4 if dtype == torch.float32 else 8
            for name, y in (("few", x.masked_fill(~few, -INF)), ("one place", x.masked_fill(at // per % 64 == 63, -INF)),
                            ("not finite", x.masked_fill(few, float("nan")).masked_fill(few.roll(5, 1), INF)),
                            ("steps", (x * 2).round() / 2)):
                y = y.to(dtype)
                for top in sorted({1, min(16, vocab), min(64, vocab)}):
                    announce("%s %s rows=%d top=%d" % (name, dtype, rows, top))
                    assert torch.equal(ops.token_log_probs(y, top=top)[4], order(y, top)), (name, dtype, rows, top)


def test_shapes():
    from gear_amd import ops
    announce("logits: shapes")
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(4, 5, 6, 50, generator=g, device="cuda")[:, :, 2]  # [4, 5, 50], rows at one stride
    tokens = torch.randint(0, 50, (4, 5), generator=g, device="cuda")
    outs = ops.token_log_probs(x, tokens, top=2)
    flat = ops.token_log_probs(x.reshape(20, 50), tokens.flatten(), top=2)
    for a, b, more in zip(outs, flat, ((), (), (), (2,), (2,))):
        assert a.shape == (4, 5) + more and torch.equal(a.reshape(b.shape), b)
    one = ops.token_log_probs(x[0, 0], tokens[0, 0], top=2)
    assert one[0].shape == () and one[4].shape == (2,) and torch.equal(one[4], outs[4][0, 0])
    loss, _ = ops.distill(x, outs[4], outs[3])
    assert loss.shape == (4, 5) and float(loss.min()) > 0  # (a teacher renormalised over two says less than the student)
    assert ops.token_log_probs(x[:0], tokens[:0], top=3)[4].shape == (0, 5, 3)
    assert ops.token_log_probs_backward(None, None, x, None, outs[2], None).abs().sum() == 0
    row = x[0, 0].expand(7, 50)  # one row for all
    assert torch.equal(ops.token_log_probs(row)[1], outs[1][0, 0].expand(7))


@pytest.mark.parametrize("vocab", [6, 600, 2600])
def test_gradients_against_differences(vocab):
    from gear_amd import sequence
    announce("logits: gradients against differences %d" % vocab)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn(3, vocab, generator=g, device="cuda") * 2)
    x[1, 2] = -INF
    x.requires_grad_()
    tokens, best = torch.tensor([1, 0, -1], device="cuda"), torch.tensor([[0, 3], [1, 1], [4, -1]], device="cuda")
    t = torch.tensor([[0.5, -1.0], [0.0, 0.3], [2.0, 1.0]], device="cuda")
    a, b, c = torch.randn(3, 3, generator=g, device="cuda")
    logp, entropy = sequence.token_log_probs(x, tokens, scale=0.8)[:2]
    ((logp * a).sum() + (entropy * b).sum() + (sequence.distill(x, best, t, scale=0.8) * c).sum()).backward()

    def f(x):
        z = x * float(torch.tensor(0.8))
        l = torch.log_softmax(z, -1)
        p = torch.exp(l)
        h = -(p * torch.where(p > 0, l, 0.0)).sum(-1)
        q, _, _ = teacher(best, t, vocab)
        d = (torch.special.xlogy(q, q) - q * l.gather(1, best.clamp(min=0))).sum(-1)
        live = torch.tensor([1.0, 1.0, 0.0], dtype=torch.float64, device="cuda")
        return ((torch.stack([l[0, 1], l[1, 0], 0 * l[2, 0]]) * a.double() + h * live * b.double()) + d * c.double()).sum()

    h = 1e-5
    for i in range(3):
        for j in list(range(6)) + [vocab - 1]:
            up, down = x.detach().double().clone(), x.detach().double().clone()
            up[i, j] += h
            down[i, j] -= h
            if (i, j) == (1, 2):
                continue
            assert abs(float((f(up) - f(down)) / (2 * h)) - float(x.grad[i, j])) < 1e-5
    assert float(x.grad[1, 2]) == 0


def test_autograd_forms():
    """What is not differentiable, and gradients as autograd hands them on."""
    from gear_amd import ops, sequence
    announce("logits: autograd")
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 90, generator=g, device="cuda").bfloat16().requires_grad_()
    tokens = torch.randint(0, 90, (4,), generator=g, device="cuda")
    outs = sequence.token_log_probs(x, tokens, top=2)
    assert [t.requires_grad for t in outs] == [True, True, False, False, False]
    outs[0].sum().backward()  # an expanded gradient, and none of the entropy
    want = ops.token_log_probs_backward(torch.ones(4, device="cuda"), None, x.detach(), tokens, outs[2], outs[1].detach())
    assert torch.equal(x.grad, want)
    x.grad = None
    sequence.token_log_probs(x)[1].mean().backward()
    assert x.grad is not None and bool(torch.isfinite(x.grad).all())
    with pytest.raises(ValueError, match="top_logits have no gradient"):
        sequence.distill(x, outs[4], outs[3].clone().requires_grad_())
