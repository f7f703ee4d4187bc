"""The model of tokens as other programs use it."""
import pytest

from conftest import announce

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _windows(vocab, step, batch=6, steps=7, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(0, vocab, (batch, steps, step), generator=g, device="cuda")
    mask, done = torch.ones(batch, steps, dtype=torch.uint8, device="cuda"), torch.zeros(batch, steps, dtype=torch.uint8, device="cuda")
    mask[0, :3], mask[1, 5:], done[2, 4] = 0, 0, 1
    return tokens, mask, done


@pytest.mark.parametrize("parameters", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16])
def test_autocast(cast, parameters):
    """Under autocast: the model's own numbers but for roundings, gradients in the parameters' type, and steps of rollouts."""
    from gear_amd.sequence import Rollouts, TokenModel, distill
    announce("token model under autocast %s %s" % (cast, parameters))
    torch.manual_seed(4)
    model = TokenModel(300, 4, width=64, heads=2, kv_heads=1, dtype=torch.float16).cuda().to(parameters)
    tokens, mask, done = _windows(300, 4)
    # (one teacher's say for both: which tokens are its best five jumps where two are nearly as probable)
    with torch.no_grad():
        best = model.log_probs(tokens, mask, done, top=5)

    def grads():
        model.zero_grad()
        logp, entropy = model.log_probs(tokens, mask, done)[:2]
        loss = distill(model(tokens, mask, done), best[4], best[3])
        (-(logp.sum() + 0.1 * entropy.sum()) / 42 + loss.sum() / 42).backward()
        return logp.detach(), entropy.detach(), [p.grad for p in model.parameters()]

    want = grads()
    with torch.autocast("cuda", dtype=cast):
        assert model(tokens, mask, done).dtype == cast
        got = grads()
        assert bool(torch.isfinite(model.distilled(model, tokens, mask, done, count=5)).all())
    # two layers of operands of O(1): the roundings of the coarsest type there is (as test_model_against_torch has it)
    unit = max(torch.finfo(cast).eps, torch.finfo(parameters).eps)
    assert float((got[0] - want[0]).abs().max()) < 32 * unit and float((got[1] - want[1]).abs().max()) < 32 * unit
    for (n, p), a, b in zip(model.named_parameters(), got[2], want[2]):
        assert a.dtype == parameters and float((a.float() - b.float()).norm()) <= 32 * unit * float(b.float().norm()) + 1e-6, n
    steps, outs = tokens[3:, 0], []
    for enabled in (False, True):
        with torch.autocast("cuda", dtype=cast, enabled=enabled):
            outs.append(model.step(Rollouts(model, 3, 8), steps[:, :3], top=64))
    assert float((outs[0][0] - outs[1][0]).abs().max()) < 32 * unit
    # (the k-th largest of numbers that are off by no more than that is off by no more)
    assert float((outs[0][1] - outs[1][1]).abs().max()) < 32 * unit


def test_norms_are_modules():
    """Hooks of the norms run, as those of any module, in windows and in steps; their names and states are nn.LayerNorm's."""
    from gear_amd.sequence import Rollouts, TokenModel
    announce("token model: hooks of norms")
    model = TokenModel(50, 3, width=64, heads=2, kv_heads=1, layers=2).cuda()
    norms = {n: m for n, m in model.named_modules() if isinstance(m, torch.nn.LayerNorm)}
    assert sorted(norms) == ["blocks.0.before", "blocks.0.between", "blocks.1.before", "blocks.1.between", "norm"]
    tokens, mask, done = _windows(50, 3)
    want = model.log_probs(tokens, mask, done)
    before, after = [], []
    for n, m in norms.items():
        m.register_forward_pre_hook(lambda module, args, n=n: before.append(n))
        m.register_forward_hook(lambda module, args, out, n=n: after.append(n))
    got = model.log_probs(tokens, mask, done)
    order = ["blocks.0.before", "blocks.0.between", "blocks.1.before", "blocks.1.between", "norm"]
    assert before == after == order and torch.equal(got[0], want[0])
    model.step(Rollouts(model, 6, 4), tokens[:, 0, :2])
    assert before == after == order * 2
    # a hook's result takes the place of the norm's
    model.norm.register_forward_hook(lambda module, args, out: (out[0] * 0, out[1]))
    assert float(model(tokens, mask, done).detach().abs().max()) == 0
    # the states that were saved before are those of today
    other = TokenModel(50, 3, width=64, heads=2, kv_heads=1, layers=2).cuda()
    other.load_state_dict(model.state_dict())
    assert torch.equal(other.log_probs(tokens, mask, done)[0], want[0])
    # other modules in their places: sums and norms of torch, in 32 bits a few roundings away
    for block in other.blocks:
        block.before, block.between = torch.nn.LayerNorm(64).cuda(), torch.nn.LayerNorm(64).cuda()
    other.norm = torch.nn.LayerNorm(64).cuda()
    # (attention in bfloat16: a rounding of its operands that falls the other way is 2^-8 of one)
    assert float((other.log_probs(tokens, mask, done)[0] - want[0]).detach().abs().max()) < 32 * 2.0 ** -8
