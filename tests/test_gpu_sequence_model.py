"""The differentiable forms of the operators, and the model that uses them together: training over the loader's windows
and rollouts from caches."""
import importlib.util
import os

import pytest

from conftest import ROOT, announce
from sequence_reference import Attention, worst

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("train_sequence_model", os.path.join(ROOT, "examples", "train_sequence_model.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_gradients_through_autograd():
    """The same numbers as the explicit calls, for gradients as autograd hands them on: expanded, transposed, of a leaf that
    is used twice."""
    from gear_amd import ops, sequence
    g = torch.Generator(device="cuda").manual_seed(0)
    announce("autograd of the sequence operators")
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    qkv = draw(2, 50, 8, 32).requires_grad_()
    wq, wk = (torch.rand(32, generator=g, device="cuda").requires_grad_() for _ in range(2))
    pos = torch.arange(50, dtype=torch.int32, device="cuda").expand(2, 50)[..., None].contiguous()
    freqs = ops.rotation_freqs((16,))
    lo, hi, _ = ops.token_ranges(torch.ones(2, 50, dtype=torch.uint8, device="cuda"))
    q, k, v = qkv.split([4, 2, 2], 2)
    rq, rk = sequence.norm_rotate(q, k, pos, freqs, (16,), wq, wk)
    out = sequence.range_attention(rq, rk, v, lo, hi, cap=5.0)
    out.sum().backward()  # an expanded gradient
    dout = torch.ones_like(out)
    o, lse = ops.range_attention(rq.detach(), rk.detach(), v.detach(), lo, hi, cap=5.0)
    drq, drk, dv = ops.range_attention_backward(dout, rq.detach(), rk.detach(), v.detach(), o, lse, lo, hi, cap=5.0)
    dq, dk, dwq, dwk = ops.norm_rotate_backward(drq, drk, q.detach(), k.detach(), pos, freqs, (16,), wq.detach(), wk.detach())
    assert torch.equal(qkv.grad, torch.cat([dq, dk, dv], 2))
    assert torch.equal(wq.grad, dwq) and torch.equal(wk.grad, dwk)
    # and the attention's against the definition, from a transposed gradient
    x = [t.detach().clone().requires_grad_() for t in (rq, rk, v)]
    gt = draw(2, 4, 50, 32)
    sequence.range_attention(*x, lo, hi).transpose(1, 2).backward(gt)
    ref = Attention(*(t.detach() for t in x), lo, hi, dout=gt.transpose(1, 2))
    for t, name in zip(x, ("dq", "dk", "dv")):
        assert worst(t.grad, getattr(ref, name), getattr(ref, name + "_bound")) <= 1
    with pytest.raises(ValueError, match="slopes have no gradient"):
        sequence.range_attention(*x, lo, hi, slopes=torch.ones(4, device="cuda", requires_grad=True))


def test_padding_and_episodes_do_not_matter_to_a_token():
    """A window's outputs are those of its documents taken alone, wherever they lie and whatever the padding holds."""
    from gear_amd.sequence import WindowModel
    torch.manual_seed(0)
    announce("documents alone and together")
    model = WindowModel(5, 3, width=64, heads=2, kv_heads=1, dtype=torch.float16).cuda()
    obs, act = torch.randn(1, 20, 5, device="cuda"), torch.randn(1, 20, 3, device="cuda")
    mask, done = torch.ones(1, 20, dtype=torch.uint8, device="cuda"), torch.zeros(1, 20, dtype=torch.uint8, device="cuda")
    mask[0, :4], done[0, 10] = 0, 1
    whole = model(obs, act, mask, done)
    obs[0, :4], act[0, :4] = 1e4, -1e4
    again = model(obs, act, mask, done)
    assert torch.equal(whole[0, 4:], again[0, 4:])
    # (other tiles, other sums: f16 rounding of operands of O(1), 2 layers)
    for a, b in ((4, 11), (11, 20)):
        alone = model(obs[:, a:b], act[:, a:b], mask[:, a:b], done[:, a:b] * 0)
        assert float((alone - whole[:, a:b]).detach().abs().max()) < 64 * 2.0 ** -11


def test_training_and_rollouts():
    """The example's model learns its policy from windows, and a rollout, token by token from caches, predicts what the model
    predicts over the whole window."""
    from gear_amd.sequence import Rollouts, WindowModel
    example = _example()
    torch.manual_seed(0)
    announce("the example: training")
    model = WindowModel(example.OBSERVATION, example.ACTION, dtype=torch.float16).cuda()
    losses = example.train(model, example.loader(example.dataset(64, key=os.getpid() + 77), 128), 60)
    assert bool(torch.isfinite(losses).all()) and float(losses[-5:].mean()) < 0.5 * float(losses[:5].mean())
    announce("the example: rollouts")
    steps, batch = 17, 9
    obs, act = torch.randn(batch, steps, example.OBSERVATION, device="cuda"), torch.rand(batch, steps, example.ACTION, device="cuda")
    with torch.no_grad():
        ones = torch.ones(batch, steps, dtype=torch.uint8, device="cuda")
        want = model(obs, act, ones, ones * 0)
    rollouts = Rollouts(model, batch, 2 * steps)
    for t in range(steps):
        got = model.step(rollouts, obs[:, t], act[:, t - 1] if t else None)
        # (the same roundings of q, k, v; probabilities and their sums rounded in another order: 2 layers of f16)
        assert float((got - want[:, t]).abs().max()) < 64 * 2.0 ** -11
    assert rollouts.length.flatten().tolist() == [2 * steps - 1] * batch


def test_a_captured_step_replays():
    """Forward, gradients and a cache step in a HIP graph, replayed with other inputs between eager calls."""
    from gear_amd import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    q, k, v, dout = draw(3, 150, 4, 64), draw(3, 150, 2, 64), draw(3, 150, 2, 64), draw(3, 150, 4, 64)
    mask = torch.ones(3, 150, dtype=torch.uint8, device="cuda")
    pos = torch.zeros(3, 150, 1, dtype=torch.int32, device="cuda")
    freqs, w = ops.rotation_freqs((32,)), torch.ones(64, device="cuda")

    def work():
        lo, hi, p = ops.token_ranges(mask, prefix=4)
        a, b = ops.norm_rotate(q, k, p, freqs, (32,), w, w)
        out, lse = ops.range_attention(a, b, v, lo, hi, cap=9.0)
        grads = ops.range_attention_backward(dout, a, b, v, out, lse, lo, hi, cap=9.0)
        last = ops.range_attention_step(a[:, -1:], b, v, lo[:, -1:].contiguous(), hi[:, -1:].contiguous(), cap=9.0)
        return (out, lse, last) + grads + ops.norm_rotate_backward(grads[0], grads[1], q, k, p, freqs, (32,), w, w)

    announce("a captured step of the sequence operators")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = work()
    for replay in range(4):
        q.copy_(draw(3, 150, 4, 64))
        v.copy_(draw(3, 150, 2, 64))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, work()):
            assert torch.equal(a, b), replay
        torch.cuda.synchronize()


def test_rollouts_end_where_their_caches_end():
    """A step that the caches have no room for is refused before anything of it is written."""
    from gear_amd.sequence import Rollouts, WindowModel
    torch.manual_seed(0)
    announce("rollouts to the end of their caches")
    model = WindowModel(5, 3, width=64, heads=2, kv_heads=1).cuda()
    obs, act = torch.randn(4, 5, device="cuda"), torch.randn(4, 3, device="cuda")
    for tokens, steps in ((5, 3), (6, 3), (1, 1)):  # the first step is one token, every other two
        rollouts = Rollouts(model, 4, tokens)
        for t in range(steps):
            model.step(rollouts, obs, act if t else None)
        before = (rollouts.caches.clone(), rollouts.length.clone(), rollouts.time.clone())
        with pytest.raises(ValueError, match="caches of %d tokens" % tokens):
            model.step(rollouts, obs, act)
        assert all(torch.equal(a, b) for a, b in zip(before, (rollouts.caches, rollouts.length, rollouts.time)))
        rollouts.restart()  # in the same caches, which hold what the last ones left
        assert torch.equal(model.step(rollouts, obs), model.step(Rollouts(model, 4, tokens), obs))
    rollouts = Rollouts(model, 4, 0)
    with pytest.raises(ValueError, match="caches of 0 tokens"):
        model.step(rollouts, obs)


@pytest.mark.parametrize("parameters", [torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parameters_of_any_type(parameters, dtype):
    """The projections run in the parameters' type, attention in the model's: training and a rollout, the same numbers as with 32-bit
    parameters up to the roundings of the types."""
    from gear_amd.sequence import Rollouts, WindowModel
    torch.manual_seed(0)
    announce("parameters of %s, attention in %s" % (parameters, dtype))
    model = WindowModel(5, 3, width=64, heads=2, kv_heads=1, dtype=dtype).cuda()
    obs, act = torch.randn(3, 8, 5, device="cuda"), torch.randn(3, 8, 3, device="cuda")
    mask, done = torch.ones(3, 8, dtype=torch.uint8, device="cuda"), torch.zeros(3, 8, dtype=torch.uint8, device="cuda")
    want = model(obs, act, mask, done).detach()
    freqs = model.freqs.clone()
    model = model.to(parameters)
    assert model.freqs.dtype == torch.float64 and torch.equal(model.freqs, freqs)
    got = model(obs.to(parameters), act.to(parameters), mask, done)
    assert got.dtype == parameters
    # (2 layers of the coarser of both types, outputs and operands of O(1))
    unit = max(torch.finfo(parameters).eps, torch.finfo(dtype).eps)
    assert float((got.detach() - want).abs().max()) < 32 * unit
    got.square().mean().backward()
    assert all(p.grad is not None and p.grad.dtype == parameters and bool(torch.isfinite(p.grad).all()) for p in model.blocks.parameters())
    rollouts = Rollouts(model, 3, 16)
    for t in range(8):
        last = model.step(rollouts, obs[:, t].to(parameters), act[:, t - 1].to(parameters) if t else None)
        assert float((last - got[:, t]).detach().abs().max()) < 32 * unit
