"""Per-head norms with the position rotation, forward, backward and into a cache, against 64 bits."""
import pytest

from conftest import announce
from sequence_reference import UNIT, norm_rotate

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SECTIONS = {16: [8], 32: [3, 0, 13], 48: [24], 64: [10], 80: [16, 12, 12], 96: [0], 128: [24, 20, 20], 144: [72],
            256: [100, 1, 20, 7]}


def _inputs(B, T, Hq, Hk, D, dtype, seed, late=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, T, Hq + 2 * Hk, D, generator=g, device="cuda").mul(3).to(dtype)
    sections = SECTIONS[D]
    freqs = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in sections]).cuda()
    pos = torch.randint(-2 ** 31 if late else 0, 2 ** 31 - 1 if late else 1000, (B, T, len(sections)), generator=g,
                        device="cuda", dtype=torch.int64).int()
    wq, wk = 1 + 0.3 * torch.randn(2, D, generator=g, device="cuda")
    return x[:, :, :Hq], x[:, :, Hq:Hq + Hk], x[:, :, Hq + Hk:], pos, freqs, sections, wq, wk, g


def _bound(ref, dtype, size):
    """One rounding to the type; in 32 bits the norm (a sum of squares: at most 16 additions deep), its root, two products,
    the sines (4 units) and a sum of two products: 32 units of the pair's size."""
    return UNIT[dtype] * ref.abs() * (0 if dtype == torch.float32 else 1) + 32 * 2.0 ** -24 * size + \
        (2.0 ** -25 if dtype == torch.float16 else 0)


def _pair_size(y):
    a, b = y.abs().chunk(2, -1)
    return torch.cat([a + b, a + b], -1)


@pytest.mark.parametrize("D", sorted(SECTIONS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_forward_and_backward(D, dtype):
    from gear_amd import ops
    for B, T, Hq, Hk, late in ((1, 1, 1, 1, False), (3, 37, 6, 2, False), (2, 5, 3, 3, True), (1, 2100, 5, 1, False)):
        q, k, _, pos, freqs, sections, wq, wk, g = _inputs(B, T, Hq, Hk, D, dtype, D + T, late)
        how = (pos, freqs, sections, wq, wk)
        announce("norm_rotate %s B=%d T=%d heads=%d/%d D=%d" % (dtype, B, T, Hq, Hk, D))
        gq = torch.randn(B, T, Hq, D, generator=g, device="cuda").to(dtype)
        # (a gradient that comes transposed from its consumer)
        gk = torch.randn(B, Hk, T, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
        outs = ops.norm_rotate(q, k, *how, eps=1e-5)
        grads = ops.norm_rotate_backward(gq, gk, q, k, *how, eps=1e-5)
        for x, w, got, gy, dx, dw in ((q, wq, outs[0], gq, grads[0], grads[2]), (k, wk, outs[1], gk, grads[1], grads[3])):
            x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
            y = norm_rotate(x64, w64, pos, freqs, sections, 1e-5)
            n = x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + 1e-5)
            size = _pair_size((n * w64).detach())
            assert got.dtype == dtype and got.is_contiguous()
            assert bool(((got.double() - y).abs() <= _bound(y.detach(), dtype, size)).all())
            rx, rw = torch.autograd.grad(y, (x64, w64), gy.double())
            # dx: r (h - n mean(h n)): the size of what is subtracted, and its mean over the row
            h = (_pair_size(gy.double()) * w64.abs()).detach()
            r = (n / torch.where(x64 == 0, 1.0, x64)).abs().amax(-1, keepdim=True).detach()
            n = n.detach()
            most = r * (h + n.abs() * (h * n.abs()).mean(-1, keepdim=True))
            assert bool(((dx.double() - rx).abs() <= _bound(rx, dtype, most)).all())
            # dw: a sum of rows in 32 bits; its order is a tree over at most 2^8 partial sums of running ones
            rows = _pair_size(gy.double()) * n.abs()
            assert bool(((dw.double() - rw).abs() <= 32 * 2.0 ** -24 * rows.sum((0, 1, 2)) + 1e-30).all())


def test_gradient_against_differences():
    from gear_amd import ops
    q, k, _, pos, freqs, sections, wq, wk, g = _inputs(1, 2, 2, 1, 32, torch.float32, 5)
    gq, gk = torch.randn(1, 2, 2, 32, generator=g, device="cuda"), torch.randn(1, 2, 1, 32, generator=g, device="cuda")
    announce("norm_rotate: differences")
    dq, dk, dwq, dwk = ops.norm_rotate_backward(gq, gk, q, k, pos, freqs, sections, wq, wk)

    def value(q, k, wq, wk):
        a, b = ops.norm_rotate(q.contiguous(), k.contiguous(), pos, freqs, sections, wq, wk)
        return float((a.double() * gq.double()).sum() + (b.double() * gk.double()).sum())

    # a central difference over 2h of a value that is off by at most 64 units of 32 bits of its terms' sizes, and by
    # h^2/6 of the third derivative (of the order of the terms over the smallest |row|^2)
    h = 2.0 ** -5
    size = float(gq.abs().sum() + gk.abs().sum()) * 4
    tol = 64 * 2.0 ** -24 * size / h + h * h * size
    args = [q.contiguous(), k.contiguous(), wq, wk]
    for i, d in enumerate((dq, dk, dwq, dwk)):
        for at in (0, 17, d.numel() - 1):
            plus, minus = [x.clone() for x in args], [x.clone() for x in args]
            plus[i].view(-1)[at] += h
            minus[i].view(-1)[at] -= h
            assert abs((value(*plus) - value(*minus)) / (2 * h) - float(d.view(-1)[at])) <= tol


@pytest.mark.parametrize("weights", ["none", "q only", "own type"])
def test_weights(weights):
    from gear_amd import ops
    q, k, _, pos, freqs, sections, wq, wk, g = _inputs(2, 9, 4, 2, 64, torch.bfloat16, 11)
    wq, wk = {"none": (None, None), "q only": (wq, None), "own type": (wq.bfloat16(), wk.bfloat16())}[weights]
    gq, gk = torch.randn(2, 9, 4, 64, generator=g, device="cuda").bfloat16(), torch.randn(2, 9, 2, 64, generator=g, device="cuda").bfloat16()
    announce("norm_rotate: weights " + weights)
    got = ops.norm_rotate(q, k, pos, freqs, sections, wq, wk)
    grads = ops.norm_rotate_backward(gq, gk, q, k, pos, freqs, sections, wq, wk)
    for x, w, y, gy, dw in ((q, wq, got[0], gq, grads[2]), (k, wk, got[1], gk, grads[3])):
        w64 = torch.ones(64, dtype=torch.float64, device="cuda") if w is None else w.double()
        w64.requires_grad_()
        ref = norm_rotate(x.double(), w64, pos, freqs, sections, 1e-6)
        assert bool(((y.double() - ref).abs() <= _bound(ref, torch.bfloat16, 8.0)).all())
        assert (dw is None) == (w is None)
        if w is not None:
            rw = torch.autograd.grad(ref, w64, gy.double())[0]
            assert dw.dtype == w.dtype
            unit = UNIT[torch.bfloat16] if w.dtype == torch.bfloat16 else 0
            assert bool(((dw.double() - rw).abs() <= unit * rw.abs() + 32 * 2.0 ** -24 * 9 * 8 * 100).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append(dtype):
    from gear_amd import ops
    for B, T, Hq, Hk, D, L in ((1, 1, 1, 1, 16, 1), (5, 3, 4, 2, 80, 40), (300, 1, 8, 8, 64, 7)):
        q, k, v, pos, freqs, sections, wq, wk, g = _inputs(B, T, Hq, Hk, D, dtype, B)
        # caches of all layers in one tensor: rows of one are apart
        caches = torch.randn(B, L, 2, 2, Hk, D, generator=g, device="cuda").to(dtype)
        k_cache, v_cache = caches[:, :, 1, 0], caches[:, :, 1, 1]
        before = caches.clone()
        slots = (torch.randint(-1, L + 1, (B, 1), generator=g, device="cuda") + torch.arange(T, device="cuda")).int()
        announce("norm_rotate_append %s B=%d T=%d D=%d" % (dtype, B, T, D))
        q_out = ops.norm_rotate_append(q, k, v, pos, freqs, sections, wq, wk, slots=slots, k_cache=k_cache, v_cache=v_cache)
        want_q, want_k = ops.norm_rotate(q, k, pos, freqs, sections, wq, wk)
        for b in range(B):
            for t in range(T):
                if 0 <= int(slots[b, t]) < L:
                    before[b, int(slots[b, t]), 1, 0] = want_k[b, t]
                    before[b, int(slots[b, t]), 1, 1] = v[b, t]
        assert torch.equal(q_out, want_q)
        assert torch.equal(caches, before)


def test_zero_rows_nan_rows_and_empty_batches():
    from gear_amd import ops
    q, k, _, pos, freqs, sections, wq, wk, _ = _inputs(2, 4, 2, 1, 32, torch.float16, 2)
    q = q.clone()
    q[0, 1] = 0
    q[1, 2, 1, 5] = float("nan")
    announce("norm_rotate: zero and NaN rows, empty batches")
    a, _ = ops.norm_rotate(q, k, pos, freqs, sections, wq, wk)
    assert not a[0, 1].any() and bool(a[1, 2, 1].isnan().all())
    a[1, 2, 1] = 0
    assert not a.isnan().any()
    for shape in ((0, 4), (2, 0)):
        e = lambda h: torch.empty(*shape, h, 32, dtype=torch.float16, device="cuda")  # noqa: E731
        p = torch.empty(*shape, len(sections), dtype=torch.int32, device="cuda")
        a, b = ops.norm_rotate(e(2), e(1), p, freqs, sections, wq, wk)
        assert a.shape == (*shape, 2, 32) and b.shape == (*shape, 1, 32)
        _, _, dwq, dwk = ops.norm_rotate_backward(e(2), e(1), e(2), e(1), p, freqs, sections, wq, wk)
        assert not dwq.any() and not dwk.any()


def test_tokens_beyond_one_launch():
    """A launch has less than 2^32 work items, 16 of them a token: 2^28 tokens and some are two."""
    from gear_amd import ops
    B, T, D = (1 << 18) + 3, 1024, 16
    announce("norm_rotate of 2^28 + 3072 tokens")
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.ones(B, T, 1, D, dtype=torch.float16, device="cuda")
    k = q[:, :, :0]
    pos = torch.zeros(B, T, 1, dtype=torch.int32, device="cuda")
    freqs = torch.full((8,), 0.5, dtype=torch.float64, device="cuda")
    for b in (0, (1 << 18) - 1, 1 << 18, B - 1):  # the border lies 16 tokens before window 2^18
        q[b] = torch.randn(T, 1, D, generator=g, device="cuda").half()
        pos[b, :, 0] = torch.arange(T, dtype=torch.int32, device="cuda")
    out, _ = ops.norm_rotate(q, k, pos, freqs, (8,))
    for b in (0, (1 << 18) - 1, 1 << 18, B - 1):
        want, _ = ops.norm_rotate(q[b:b + 1], k[b:b + 1], pos[b:b + 1].contiguous(), freqs, (8,))
        assert torch.equal(out[b:b + 1], want)
    ones = torch.ones(1, dtype=torch.float16, device="cuda")
    for b in range(1, B, 8192):
        if b not in (0, (1 << 18) - 1, 1 << 18, B - 1):
            assert bool((out[b] - ones).abs().max() <= 2.0 ** -10)


def test_gradient_against_differences_in_64_bits():
    """The gradients against central differences of the definition in 64 bits: h = 1e-4, the differences are off by h^2 / 6 of a third
    derivative (rows of about 3 an element, weights of about 1: below 16 a unit of the gradient that comes in) and 1e-16 / h of
    the value, the gradients by 64 units of 32 bits of what is summed.  Every element, and the largest are a hundred times the
    bound and more."""
    from gear_amd import ops
    q, k, _, pos, freqs, sections, wq, wk, g = _inputs(2, 3, 2, 1, 32, torch.float32, 5)
    gq, gk = torch.randn(2, 3, 2, 32, generator=g, device="cuda"), torch.randn(2, 3, 1, 32, generator=g, device="cuda")
    announce("norm_rotate: differences in 64 bits")
    grads = ops.norm_rotate_backward(gq, gk, q, k, pos, freqs, sections, wq, wk)
    args = [x.double().contiguous() for x in (q, k, wq, wk)]

    def value(q, k, wq, wk):
        a, b = norm_rotate(q, wq, pos, freqs, sections, 1e-6), norm_rotate(k, wk, pos, freqs, sections, 1e-6)
        return float((a * gq.double()).sum() + (b * gk.double()).sum())

    h = 1e-4
    size = float(gq.abs().sum() + gk.abs().sum())
    tol = h * h / 6 * 16 * float(gq.abs().max()) * 32 + 1e-15 * size * 4 / h + 64 * 2.0 ** -24 * float(gq.abs().amax()) * 32
    for i, grad in enumerate(grads):
        slopes = []
        for at in range(grad.numel()):
            plus, minus = [x.clone() for x in args], [x.clone() for x in args]
            plus[i].view(-1)[at] += h
            minus[i].view(-1)[at] -= h
            slopes.append((value(*plus) - value(*minus)) / (2 * h))
        slopes = torch.tensor(slopes, dtype=torch.float64, device="cuda").view(grad.shape)
        assert float(slopes.abs().max()) > 100 * tol
        assert float((grad.double() - slopes).abs().max()) <= tol
