"""Attention over ranges of keys, forward, backward and over caches, against 64 bits."""
import itertools
import math

import pytest

from conftest import announce
from sequence_reference import UNIT, Attention, worst

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def _rows(g, B, T, H, D, dtype, scale=1.0):
    return (torch.randn(B, T, H, D, generator=g, device="cuda") * scale).to(dtype)


def _masks(kind, B, T, S, g):
    i = torch.arange(T, device="cuda").expand(B, T) + S - T
    zero = torch.zeros_like(i)
    if kind == "causal":
        lo, hi = zero, i + 1
    elif kind == "all":
        lo, hi = zero, zero + S
    elif kind == "documents":  # runs of 1 to 40 tokens, causal, empty rows between some
        cut = torch.rand(B, T, generator=g, device="cuda") < 0.08
        lo = torch.cummax(torch.where(cut, i, zero), 1).values
        gone = torch.rand(B, T, generator=g, device="cuda") < 0.15
        hi = torch.where(gone, lo, i + 1)
    elif kind == "prefix":
        lo, hi = zero, torch.maximum(i + 1, zero + S // 3)
    elif kind == "band":
        lo, hi = i - 20, i + 5  # reaches below 0 and beyond S
    elif kind == "any":  # no order between rows at all
        a, b = torch.randint(-5, S + 6, (2, B, T), generator=g, device="cuda")
        lo, hi = a, b
    else:  # nothing
        lo, hi = zero + 3, zero + 3
    return lo.int().contiguous(), hi.int().contiguous()


def _check(B, T, S, H, HK, D, dtype, mask, cap=0.0, slopes=False, scale=None, seed=0, train=True):
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = _rows(g, B, T, H, D, dtype, 1.5)
    k, v = _rows(g, B, S, 2 * HK, D, dtype, 1.5).split(HK, 2)  # side by side: not contiguous
    lo, hi = _masks(mask, B, T, S, g)
    form = dict(cap=cap, scale=scale, slopes=torch.rand(H, generator=g, device="cuda") if slopes else None)
    announce("attention %s B=%d T=%d S=%d heads=%d/%d D=%d %s cap=%g slopes=%s" % (dtype, B, T, S, H, HK, D, mask, cap, slopes))
    out, lse = ops.range_attention(q, k, v, lo, hi, **form)
    dout = _rows(g, B, H, T, D, dtype).transpose(1, 2) if train else None
    ref = Attention(q, k, v, lo, hi, dout=dout, **form)
    assert out.is_contiguous() and worst(out, ref.out, ref.out_bound) <= 1
    assert worst(lse, ref.lse, ref.lse_bound) <= 1
    if not train:
        return
    dq, dk, dv = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi, **form)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert got.dtype == dtype and got.is_contiguous()
        assert worst(got, getattr(ref, name), getattr(ref, name + "_bound")) <= 1, name
    again = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi, **form)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", ["causal", "all", "documents", "prefix", "band", "any", "nothing"])
def test_masks(mask, dtype):
    for (T, S), (cap, slopes) in itertools.product(((1, 1), (5, 70), (130, 130), (200, 333)), ((0.0, False), (4.0, True))):
        _check(2, T, S, 4, 2, 64, dtype, mask, cap, slopes, seed=T + S)


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("heads", [(1, 1), (6, 2), (8, 1)])
def test_sizes(D, heads):
    for dtype in TYPES:
        for T in (31, 32, 33, 63, 65, 128, 129):
            _check(2, T, T, heads[0], heads[1], D, dtype, "documents", seed=D + T)


def test_many_queries_and_keys():
    _check(1, 1500, 1500, 2, 1, 128, torch.bfloat16, "causal", seed=1)
    _check(1, 3000, 3000, 1, 1, 32, torch.float16, "documents", cap=10.0, seed=2)
    _check(1, 4200, 70, 2, 2, 64, torch.float16, "all", seed=3)
    _check(3, 90, 5000, 3, 3, 48, torch.bfloat16, "any", slopes=True, seed=4)
    _check(70, 90, 90, 2, 2, 64, torch.bfloat16, "causal", seed=5)


def test_scale_and_large_scores():
    """Scores of hundreds: the maximum is taken off before the exponent."""
    _check(2, 100, 100, 2, 2, 64, torch.float16, "causal", scale=3.0, seed=6)
    _check(2, 100, 100, 2, 2, 64, torch.bfloat16, "causal", scale=1e-3, seed=7)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_no_range_reaches_is_not_looked_at(dtype):
    """Padding as torch.empty leaves it: NaN and infinities in keys nobody sees, in queries that see nothing and in
    their gradients."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(8)
    for T, pad in ((90, 30), (200, 64), (300, 131)):
        q, k, v, dout = (_rows(g, 2, T, 4, 64, dtype) for _ in range(4))
        i = torch.arange(T, device="cuda").expand(2, T)
        lo = torch.full_like(i, pad).int()
        hi = torch.where(i < pad, 0, i + 1).int()
        clean = [x.clone() for x in (q, k, v, dout)]
        for x in clean:
            x[:, :pad] = 0
        for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
            for x in (q, k, v, dout):
                x[:, :pad] = bad
            announce("padding of %s, T=%d, %s" % (bad, T, dtype))
            out, lse = ops.range_attention(q, k, v, lo, hi)
            want, want_lse = ops.range_attention(*clean[:3], lo, hi)
            assert torch.equal(out, want) and torch.equal(lse, want_lse)
            assert not out[:, :pad].any() and bool((lse[..., :pad] == -float("inf")).all())
            got = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi)
            for a, b in zip(got, ops.range_attention_backward(clean[3], *clean[:3], want, want_lse, lo, hi)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_some_rows_see_does_not_reach_the_others(dtype, bad):
    """A key (or a query and its gradient) that is not finite: rows that see it are NaN or infinite, the others as if it
    were not there."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(14)
    for T, H, HK, D, cap in ((90, 2, 2, 64, 0.0), (90, 4, 2, 48, 6.0), (300, 2, 1, 128, 0.0), (200, 2, 2, 32, 6.0)):
        q, k, v, dout = (_rows(g, 2, T, h, D, dtype) for h in (H, HK, HK, H))
        form = dict(cap=cap, slopes=torch.rand(H, generator=g, device="cuda") * 0.1 if cap else None)
        lo, hi = _masks("causal", 2, T, T, g)
        ref = Attention(q, k, v, lo, hi, dout=dout, **form)
        at = 2 * T // 3 + 5
        announce("%s at %d of %d, %s, D=%d" % (bad, at, T, dtype, D))
        # a key: queries before it do not see it
        k2, v2 = k.clone(), v.clone()
        k2[0, at, :, 3] = bad
        v2[0, at] = bad
        out, lse = ops.range_attention(q, k2, v2, lo, hi, **form)
        same = torch.ones(2, T, dtype=torch.bool, device="cuda")
        same[0, at:] = False
        pick = lambda x: x[same]  # noqa: E731
        assert worst(pick(out), pick(ref.out), pick(ref.out_bound)) <= 1
        assert worst(lse.transpose(1, 2)[same], ref.lse.transpose(1, 2)[same], ref.lse_bound.transpose(1, 2)[same]) <= 1
        assert not torch.isfinite(out[0, at:]).all(-1).any()
        dq = ops.range_attention_backward(dout, q, k2, v2, out, lse, lo, hi, **form)[0]
        assert worst(pick(dq), pick(ref.dq), pick(ref.dq_bound)) <= 1
        # a query and its gradient: keys behind it are not seen by it
        q2, dout2 = q.clone(), dout.clone()
        q2[1, at], dout2[1, at] = bad, bad
        out, lse = ops.range_attention(q2, k, v, lo, hi, **form)
        dq, dk, dv = ops.range_attention_backward(dout2, q2, k, v, out, lse, lo, hi, **form)
        same[:] = True
        same[1, at] = False
        assert worst(pick(out), pick(ref.out), pick(ref.out_bound)) <= 1
        assert worst(pick(dq), pick(ref.dq), pick(ref.dq_bound)) <= 1
        same[:] = True
        same[1, :at + 1] = False
        assert worst(pick(dk), pick(ref.dk), pick(ref.dk_bound)) <= 1
        assert worst(pick(dv), pick(ref.dv), pick(ref.dv_bound)) <= 1
        assert not torch.isfinite(dv[1, :at + 1]).any()
        # over caches: the newest of three tokens sees one key more
        new = hi[:, at - 2:at + 1].contiguous()
        out = ops.range_attention_step(q[:, at - 2:at + 1], k2, v2, lo[:, :3].contiguous(), new, **form)
        assert worst(out[0, :2], ref.out[0, at - 2:at], ref.out_bound[0, at - 2:at]) <= 1
        assert not torch.isfinite(out[0, 2]).all(-1).any()
        assert worst(out[1], ref.out[1, at - 2:at + 1], ref.out_bound[1, at - 2:at + 1]) <= 1


def test_gradient_against_differences():
    """f16 inputs, a step of 2^-4: the value is a sum of B*T*H*D products of out (rounded: 2^-11 of its size)."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k, v, dout = (_rows(g, 1, 6, 2, 16, torch.float16) for _ in range(4))
    lo, hi = _masks("causal", 1, 6, 6, g)
    form = dict(cap=3.0, slopes=torch.tensor([0.1, 0.4], device="cuda"))
    announce("attention: differences")
    out, lse = ops.range_attention(q, k, v, lo, hi, **form)
    grads = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi, **form)
    h = 2.0 ** -4
    for i, grad in enumerate(grads):
        for at in (0, 40, 100, 191):
            values = []
            for sign in (1, -1):
                args = [x.clone() for x in (q, k, v)]
                args[i].view(-1)[at] += sign * h
                step = float(args[i].view(-1)[at]) - float((q, k, v)[i].view(-1)[at])
                values.append((step, Attention(*args, lo, hi, **form).out.flatten() @ dout.double().flatten()))
            slope = float((values[0][1] - values[1][1]) / (values[0][0] - values[1][0]))
            # the difference's own error: h^2/6 of the third derivative (scores of O(1): below 4 a term); the gradient's: its bound
            ref = Attention(q, k, v, lo, hi, dout=dout, **form)
            name = ("dq", "dk", "dv")[i]
            bound = float(getattr(ref, name + "_bound").flatten()[at])
            assert abs(float(grad.view(-1)[at]) - slope) <= bound + h * h / 6 * 4 * float(dout.abs().sum()) / 6


@pytest.mark.parametrize("dtype", TYPES)
def test_step_over_caches(dtype):
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(10)
    for B, T, L, H, HK, D in ((1, 1, 1, 1, 1, 16), (3, 1, 33, 4, 4, 64), (2, 3, 700, 6, 2, 80), (5, 2, 257, 32, 2, 128),
                              (2, 1, 40000, 16, 2, 64), (1, 70, 300, 4, 4, 32), (300, 4, 90, 3, 3, 48)):
        q, k, v = _rows(g, B, T, H, D, dtype, 1.5), _rows(g, B, L, HK, D, dtype, 1.5), _rows(g, B, L, HK, D, dtype, 1.5)
        hi = torch.randint(0, L + 1, (B, 1), generator=g, device="cuda") - torch.arange(T, device="cuda").flip(0)
        lo = (torch.rand(B, 1, generator=g, device="cuda") * 0.5 * hi.clamp(min=0)).long().expand(B, T).clone()
        lo[0] = -3
        hi[0, -1] = L + 9
        lo, hi = lo.int().contiguous(), hi.int().contiguous()
        # beyond what is filled a cache holds anything
        at = torch.arange(L, device="cuda")
        free = (at[None] >= hi.amax(1, keepdim=True))[:, :, None, None]
        k, v = torch.where(free, float("nan"), k), torch.where(free, float("inf"), v)
        for cap, slopes in ((0.0, False), (5.0, True)):
            form = dict(cap=cap, slopes=torch.rand(H, generator=g, device="cuda") * 0.1 if slopes else None)
            announce("step %s B=%d T=%d L=%d heads=%d/%d D=%d cap=%g" % (dtype, B, T, L, H, HK, D, cap))
            out = ops.range_attention_step(q, k, v, lo, hi, **form)
            ref = Attention(q, k, v, lo, hi, place=hi - 1, **form)
            assert worst(out, ref.out, ref.out_bound) <= 1


def test_no_keys_no_queries_no_batch():
    from gear_amd import ops
    announce("attention: empty sizes")
    for B, T, S in ((0, 4, 4), (2, 0, 4), (2, 4, 0), (2, 0, 0)):
        q, k, v = (torch.empty(B, n, 2, 32, dtype=torch.float16, device="cuda") for n in (T, S, S))
        lo, hi = torch.zeros(B, T, dtype=torch.int32, device="cuda"), torch.full((B, T), 9, dtype=torch.int32, device="cuda")
        out, lse = ops.range_attention(q, k, v, lo, hi)
        assert out.shape == q.shape and not out.any() and bool((lse == -float("inf")).all())
        dq, dk, dv = ops.range_attention_backward(q, q, k, v, out, lse, lo, hi)
        assert not dq.any() and not dk.any() and not dv.any()
        assert not ops.range_attention_step(q, k, v, lo, hi).any()


def test_rows_beyond_32_bit_offsets():
    """A cache whose last rows lie more than 2^32 elements from its first."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(12)
    announce("rows beyond 2^32 elements")
    L, stride = 70, (1 << 26) + 8
    store = torch.empty((L - 1) * stride + 64, dtype=torch.float16, device="cuda")
    far = store.as_strided((1, L, 2, 32), (0, stride, 32, 1))
    near = _rows(g, 1, L, 2, 32, torch.float16)
    far.copy_(near)
    q = _rows(g, 1, L, 2, 32, torch.float16)
    lo, hi = _masks("causal", 1, L, L, g)
    out, lse = ops.range_attention(q, near, near, lo, hi)
    got, got_lse = ops.range_attention(q, far, far, lo, hi)
    assert torch.equal(out, got) and torch.equal(lse, got_lse)
    for a, b in zip(ops.range_attention_backward(q, q, near, near, out, lse, lo, hi),
                    ops.range_attention_backward(q, q, far, far, out, lse, lo, hi)):
        assert torch.equal(a, b)
    assert torch.equal(ops.range_attention_step(q[:, -1:], near, near, lo[:, -1:].contiguous(), hi[:, -1:].contiguous()),
                       ops.range_attention_step(q[:, -1:], far, far, lo[:, -1:].contiguous(), hi[:, -1:].contiguous()))


def test_calls_on_two_streams():
    """Scratch of its own for each stream: calls in flight on two do not meet."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(13)
    announce("attention on two streams")
    sets = []
    for _ in range(2):
        q, k, v, dout = (_rows(g, 4, 300, 4, 64, torch.bfloat16) for _ in range(4))
        sets.append((q, k, v, dout) + _masks("causal", 4, 300, 300, g))
    want = []
    for q, k, v, dout, lo, hi in sets:
        out, lse = ops.range_attention(q, k, v, lo, hi)
        want.append(ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi) + (ops.range_attention_step(q[:, :1].contiguous(), k, v, lo[:, -1:].contiguous(), hi[:, -1:].contiguous()),))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(10):
        for x, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                q, k, v, dout, lo, hi = sets[x]
                out, lse = ops.range_attention(q, k, v, lo, hi)
                got[x] = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi) + (ops.range_attention_step(q[:, :1].contiguous(), k, v, lo[:, -1:].contiguous(), hi[:, -1:].contiguous()),)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_that_see_nothing_get_nothing_beside_rows_that_see_what_is_not_finite(dtype, bad):
    """Padding at the head of a window, and a key (its K, or its V) that is not finite and that every other row sees, or
    those behind it: padding gets gradients of 0 and passes none on, in one launch (T <= 128, a key head a head) and in two."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(15)
    for T, H, HK, D, cap in ((60, 2, 2, 64, 0.0), (128, 2, 2, 48, 5.0), (60, 4, 2, 64, 0.0), (200, 2, 2, 128, 0.0)):
        q, k, v, dout = (_rows(g, 2, T, h, D, dtype) for h in (H, HK, HK, H))
        pad, at = 10, 2 * T // 3
        i = torch.arange(T, device="cuda").expand(2, T)
        for sees in ("all", "causal"):
            lo = torch.where(i < pad, 0, pad).int()
            hi = torch.where(i < pad, 0, T if sees == "all" else i + 1).int()
            ref = Attention(q, k, v, lo, hi, cap=cap, dout=dout)
            for where in ("K", "V"):
                k2, v2 = k.clone(), v.clone()
                (k2 if where == "K" else v2)[0, at] = bad
                announce("padding beside %s of %s, T=%d D=%d %s %s" % (where, bad, T, D, sees, dtype))
                out, lse = ops.range_attention(q, k2, v2, lo, hi, cap=cap)
                dq, dk, dv = ops.range_attention_backward(dout, q, k2, v2, out, lse, lo, hi, cap=cap)
                assert not out[:, :pad].any() and bool((lse[..., :pad] == -float("inf")).all())
                assert torch.equal(dq[:, :pad], torch.zeros_like(dq[:, :pad]))
                assert not dk[:, :pad].any() and not dv[:, :pad].any()  # keys of padding, which nobody sees
                # rows before the key, and the other window, as if it were not there
                before = slice(0, at if sees == "causal" else pad)
                for name, got in (("out", out), ("dq", dq)):
                    want, bound = getattr(ref, name), getattr(ref, name + "_bound")
                    assert worst(got[0, before], want[0, before], bound[0, before]) <= 1
                for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
                    assert worst(got[1], getattr(ref, name)[1], getattr(ref, name + "_bound")[1]) <= 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [90, 3000])
def test_step_whose_ranges_reach_beyond_the_cache_beside_a_key_that_is_not_finite(dtype, L):
    """Two tokens, of which the second sees a key that is not finite: the first is worked out alone, and its distances count from
    the last key there is.  (In one part and in several.)"""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(16)
    B, T, H, HK, D = 2, 2, 4, 2, 64
    q, k, v = _rows(g, B, T, H, D, dtype), _rows(g, B, L, HK, D, dtype), _rows(g, B, L, HK, D, dtype)
    slopes = torch.rand(H, generator=g, device="cuda") * 0.5
    lo = torch.tensor([[50, 0], [50, 50]], dtype=torch.int32, device="cuda")
    hi = torch.tensor([[L + 7, L + 9], [L + 30, L]], dtype=torch.int32, device="cuda")
    for cap in (0.0, 5.0):
        ref = Attention(q, k, v, lo, hi, cap=cap, slopes=slopes, place=hi.clamp(max=L) - 1)
        v2 = v.clone()
        v2[0, 40:50] = float("inf")
        announce("step beyond the cache %s L=%d cap=%g" % (dtype, L, cap))
        out = ops.range_attention_step(q, k, v2, lo, hi, cap=cap, slopes=slopes)
        assert worst(out[0, 0], ref.out[0, 0], ref.out_bound[0, 0]) <= 1
        assert worst(out[1], ref.out[1], ref.out_bound[1]) <= 1
        assert not torch.isfinite(out[0, 1]).any()


@pytest.mark.parametrize("cap", [0.5, 30.0, 64.0, 65.0, 1e3, 1e5, 1e8, 1e29])
def test_capped_scores_are_as_exact_as_scores(cap):
    """A query that sees one key: its lse is its score.  q . k has one product, so that what is seen is the scale, the cap
    and the logarithm's units: a score is off by at most 16 units of 32 bits of ITSELF (its scale 1, the argument and the
    tanh 8, the exponent's factor 2, the way to base 2 and back 2; the logarithm of a sum of 1: 2e-7).  Caps up to 64 may be
    off by 2^-22 of the cap on top, 1.6e-5 at most."""
    from gear_amd import ops
    T, D = 500, 64
    announce("capped scores one by one, cap %g" % cap)
    x = torch.logspace(-4, 4, T, dtype=torch.float64, device="cuda")
    x = torch.where(torch.arange(T, device="cuda") % 2 == 0, x, -x).bfloat16()
    q, k = (torch.zeros(1, T, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q[0, :, 0, 5], k[0, :, 0, 5] = x, 1.0
    lo = torch.arange(T, dtype=torch.int32, device="cuda")[None].contiguous()
    scale = 0.125
    for slopes in (None, torch.zeros(1, device="cuda")):
        _, lse = ops.range_attention(q, k, k, lo, lo + 1, cap=cap, scale=scale, slopes=slopes)
        want = cap * torch.tanh(x.double() * scale / cap)
        near = 2.0 ** -22 * cap if cap <= 64 else 0
        assert bool(((lse[0, 0].double() - want).abs() <= 16 * 2.0 ** -24 * want.abs() + 2e-7 + near).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [30.0, 1e4, 1e6, 1e8, 1e29])
def test_large_caps(cap, dtype):
    """A cap far above the scores leaves them as they are: forward, gradients (in one launch and in two) and a step, within
    the bounds of scores without a cap (whose size is the scores', not the cap's)."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(17)
    for T, H, HK, D, slopes in ((100, 2, 2, 64, False), (300, 4, 2, 80, True)):
        q, k, v, dout = (_rows(g, 2, T, h, D, dtype, 1.5) for h in (H, HK, HK, H))
        lo, hi = _masks("documents", 2, T, T, g)
        form = dict(slopes=torch.rand(H, generator=g, device="cuda") * 0.1 if slopes else None)
        announce("cap %g, %s, T=%d" % (cap, dtype, T))
        ref, free = Attention(q, k, v, lo, hi, cap=cap, dout=dout, **form), Attention(q, k, v, lo, hi, dout=dout, **form)
        out, lse = ops.range_attention(q, k, v, lo, hi, cap=cap, **form)
        grads = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi, cap=cap, **form)
        assert worst(lse, ref.lse, free.lse_bound) <= 1
        if cap >= 1e4:  # (at 30 the probabilities, and with them the bounds, differ from those without a cap)
            for name, got in zip(("out", "dq", "dk", "dv"), (out,) + tuple(grads)):
                assert worst(got, getattr(ref, name), getattr(free, name + "_bound")) <= 1, name
        place = hi - 1
        ref, free = Attention(q, k, v, lo, hi, cap=cap, place=place, **form), Attention(q, k, v, lo, hi, place=place, **form)
        out = ops.range_attention_step(q, k, v, lo, hi, cap=cap, **form)
        assert worst(out, ref.out, ref.out_bound if cap < 1e4 else free.out_bound) <= 1


@pytest.mark.parametrize("dtype", TYPES)
def test_large_caps_that_scores_reach(dtype):
    """Scores of up to hundreds under caps of their size: tiles hold small arguments of the tanh and large ones."""
    for cap in (65.0, 200.0):
        _check(2, 100, 100, 2, 2, 64, dtype, "causal", cap, scale=3.0, seed=20)
        _check(1, 300, 300, 4, 2, 80, dtype, "documents", cap, True, scale=3.0, seed=21)


@pytest.mark.parametrize("raised", ["q", "k"])
@pytest.mark.parametrize("sizes", [(2000, 4, 2, 64), (2000, 2, 2, 128), (120, 2, 2, 64)])
@pytest.mark.parametrize("exponent", [-16, 0, 8])
def test_gradients_of_any_size_in_float16(exponent, sizes, raised):
    """Gradients are linear in dout: with dout 2^e as large (exactly) they are 2^e as large, in float16 as far as the results
    themselves can be held: a result's own step is 2^-25 at most.  q 32 times and k a 32nd as large, or the other way round,
    so that the scores are the same and dk, or dq, is large enough to be held at 2^-16."""
    from gear_amd import ops
    T, H, HK, D = sizes
    g = torch.Generator(device="cuda").manual_seed(18)
    q, k, v = (_rows(g, 1, T, h, D, torch.float16) for h in (H, HK, HK))
    q, k = (q * 32, k / 32) if raised == "q" else (q / 32, k * 32)
    dout = (torch.randn(1, T, H, D, generator=g, device="cuda") * 8).round().clamp(-16, 16) / 8  # (exact at all three sizes)
    lo, hi = _masks("all", 1, T, T, g)
    announce("gradients of float16, 2^%d, T=%d D=%d, %s raised" % (exponent, T, D, raised))
    ref = Attention(q, k, v, lo, hi, dout=dout.half())
    out, lse = ops.range_attention(q, k, v, lo, hi)
    grads = ops.range_attention_backward((dout * 2.0 ** exponent).half(), q, k, v, out, lse, lo, hi)
    for name, got in zip(("dq", "dk", "dv"), grads):
        bound = getattr(ref, name + "_bound") + 2.0 ** (-25 - exponent)
        assert worst(got.double() * 2.0 ** -exponent, getattr(ref, name), bound) <= 1, name
    # norm of the difference over the norm: a rounding of ds and one of the result, each 2^-11 / sqrt(3) at most
    # (rounding is evenly spread), delta's from out of about as much: 2^-10 holds all; what a step of 2^-25 leaves on top
    name, got = ("dk", grads[1]) if raised == "q" else ("dq", grads[0])
    want = getattr(ref, name)
    off = (got.double() * 2.0 ** -exponent - want).norm()
    assert float(off) <= 2.0 ** -10 * float(want.norm()) + 2.0 ** (-25 - exponent) * want.numel() ** 0.5


@pytest.mark.parametrize("dtype", TYPES)
def test_a_key_with_most_of_the_weight_does_not_swallow_the_others(dtype):
    """One key with nearly all of the weight, first, in the middle or last, 50 000 with 2^-25.5 of it each: their thousandth is part of
    the sum, in 32 bits.  (The bound of lse has no term for the number of keys.)"""
    from gear_amd import ops
    S, D = 50000, 32
    announce("a key with most of the weight, %s" % dtype)
    q, k, v = (torch.zeros(1, n, 1, D, dtype=dtype, device="cuda") for n in (1, S, S))
    q[..., 0] = 1.0
    lo, hi = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1, 1), S, dtype=torch.int32, device="cuda")
    for at in (0, 777, S - 1):
        k.zero_()
        k[:, at, :, 0] = 25.5 * math.log(2)
        ref = Attention(q, k, v, lo, hi, scale=1.0)
        _, lse = ops.range_attention(q, k, v, lo, hi, scale=1.0)
        assert worst(lse, ref.lse, ref.lse_bound) <= 1


def test_many_small_probabilities_in_float16():
    """One key with nearly all of the weight and v = 0, 50 000 with 2^-25.5 of it each and v = 1: together they are a thousandth.
    A probability is held to half a step, 2^-32 of the largest at most (bound), whatever its own size."""
    from gear_amd import ops
    S, D = 50000, 32
    announce("many small probabilities")
    q, k, v = (torch.zeros(1, n, 1, D, dtype=torch.float16, device="cuda") for n in (1, S, S))
    q[..., 0] = 1.0
    k[:, 777, :, 0] = 25.5 * math.log(2)
    v[...] = 1.0
    v[:, 777] = 0.0
    lo, hi = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1, 1), S, dtype=torch.int32, device="cuda")
    ref = Attention(q, k, v, lo, hi, scale=1.0)
    bound = 2 * 2.0 ** -11 * ref.out + 2.0 ** -32 * S + 1e-5 * ref.out
    out, lse = ops.range_attention(q, k, v, lo, hi, scale=1.0)
    assert worst(out, ref.out, bound) <= 1 and worst(lse, ref.lse, ref.lse_bound) <= 1
    assert worst(ops.range_attention_step(q, k, v, lo, hi, scale=1.0), ref.out, bound) <= 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
def test_a_score_of_minus_infinity_is_a_probability_of_zero(D, dtype):
    """Keys that hold -inf where every query is positive, in the first and in the last elements of a row: rows see them with
    p = 0, as the formula says, and dv of such a key is 0."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(19)
    for T, H, HK in ((70, 2, 2), (150, 4, 2)):
        for at in (1, D - 2):
            q, k, v, dout = (_rows(g, 1, T, h, D, dtype) for h in (H, HK, HK, H))
            q[..., at] = q[..., at].abs() + 0.5
            lo, hi = _masks("causal", 1, T, T, g)
            lo[:] = 0
            gone = torch.arange(T, device="cuda") % 3 == 1  # (not the first: every row keeps a key)
            k[:, gone, :, at] = -float("inf")
            without = k.clone()
            without[:, gone, :, at] = 0
            announce("scores of -inf, D=%d at %d, T=%d, %s" % (D, at, T, dtype))
            # the definition: the same keys, not seen.  In 64 bits, with the scores of those keys at -inf
            out, lse = ops.range_attention(q, k, v, lo, hi)
            ref = Attention(q, without, v, lo, hi)
            heads = lambda x: x.double().permute(0, 2, 1, 3).contiguous()  # noqa: E731
            many = lambda x: heads(x).repeat_interleave(H // HK, 1)  # noqa: E731
            s = heads(q) @ many(without).transpose(2, 3) * D ** -0.5
            i = torch.arange(T, device="cuda")
            s = s.masked_fill((i > i[:, None]) | gone, -float("inf"))
            p = torch.softmax(s, -1)
            want = (p @ many(v)).permute(0, 2, 1, 3)
            # (weights of what is left are at most what they were times the share of what went: the bound by that of |v|)
            most = float(v.abs().max())
            unit = UNIT[dtype] + 2.0 ** -24 * (8 + math.sqrt(D)) * 40
            assert worst(out, want, torch.full_like(want, 1.01 * unit * 2 * most + 2.0 ** -20)) <= 1
            assert worst(lse, torch.logsumexp(s, -1), ref.lse_bound + 1e-5) <= 1
            _, _, dv = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi)
            assert not dv[:, gone].any()
            want = (p.transpose(2, 3) @ heads(dout)).view(1, HK, H // HK, T, D).sum(2).permute(0, 2, 1, 3)
            size = (p.transpose(2, 3) @ heads(dout).abs()).view(1, HK, H // HK, T, D).sum(2).permute(0, 2, 1, 3)
            assert worst(dv, want, 1.01 * 2 * unit * size + 2.0 ** -20) <= 1
            step = ops.range_attention_step(q[:, -2:], k, v, lo[:, -2:].contiguous(), hi[:, -2:].contiguous())
            assert worst(step, (p @ many(v)).permute(0, 2, 1, 3)[:, -2:], torch.full_like(step, 1.01 * unit * 2 * most + 2.0 ** -20).double()) <= 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_dq_where_one_key_has_most_of_the_weight(cap, dtype):
    """Steep slopes: a row's last key has 0.9 and more of its weight, dp - delta is a small difference there, and a delta that
    begins from the rounded out is off by more than it.  dq is held to the roundings that it needs: of ds and of the result, each
    u / sqrt(3) of the norm at most (a rounding is evenly spread over at most 2 u), a fifth more for what keys of small weight
    and 32 bits leave.  In two launches (long rows, shared key heads, rows of 128) and in one."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(21)
    for T, H, HK, D in ((300, 2, 2, 64), (90, 4, 2, 48), (1000, 2, 1, 128), (5000, 1, 1, 32), (100, 2, 2, 64)):
        q, k, v, dout = (_rows(g, 1, T, h, D, dtype) for h in (H, HK, HK, H))
        lo, hi = _masks("causal", 1, T, T, g)
        form = dict(cap=cap, slopes=torch.linspace(4, 6, H, device="cuda"))
        announce("dq of rows with one key, %s T=%d heads=%d/%d D=%d cap=%g" % (dtype, T, H, HK, D, cap))
        out, lse = ops.range_attention(q, k, v, lo, hi, **form)
        dq, dk, _ = ops.range_attention_backward(dout, q, k, v, out, lse, lo, hi, **form)
        ref = Attention(q, k, v, lo, hi, dout=dout, **form)
        for got, want in ((dq, ref.dq), (dk, ref.dk)):
            assert float((got.double() - want).norm() / want.norm()) <= 1.2 * UNIT[dtype] * (2 / 3) ** 0.5
