"""The operators of token models together: captured, on other streams, and in the model that trains, distils and acts."""
import importlib.util
import os
import threading

import pytest

from conftest import ROOT, announce

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class _Run:
    """Tokens in, norm, logits out, and all gradients, by the explicit calls."""

    def __init__(self, seed, rows=600, vocab=2500, width=72, dtype=torch.bfloat16):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        draw = lambda *s: torch.randn(*s, generator=self.g, device="cuda").to(dtype)  # noqa: E731
        self.rows, self.vocab, self.width = rows, vocab, width
        self.tokens = torch.randint(-1, vocab, (rows,), generator=self.g, device="cuda")
        self.table, self.more, self.head = draw(vocab, width), draw(rows, width), draw(width, vocab)
        self.w, self.b = torch.rand(2, width, generator=self.g, device="cuda")
        self.dl, self.de = torch.randn(2, rows, generator=self.g, device="cuda")

    def renew(self):
        self.tokens.copy_(torch.randint(-1, self.vocab, (self.rows,), generator=self.g, device="cuda"))
        self.more.copy_(torch.randn(self.rows, self.width, generator=self.g, device="cuda"))

    def __call__(self):
        from gear_amd import ops
        x = ops.embed_tokens(self.tokens, self.table, scale=2.0)
        y, u = ops.layer_norm(self.more, self.w, self.b, residual=x)
        logits = y @ self.head
        few = logits[:3]  # (rows in parts, and their join)
        outs = ops.token_log_probs(logits, self.tokens, top=5)
        step = ops.token_log_probs(few, top=5)
        loss, lse = ops.distill(logits, outs[4], outs[3])
        dz = ops.token_log_probs_backward(self.dl, self.de, logits, self.tokens, outs[2], outs[1])
        dd = ops.distill_backward(self.dl, logits, outs[4], outs[3], lse)
        dx, dw, db = ops.layer_norm_backward(dz @ self.head.t().contiguous(), u, self.w, self.b, dsum=y)
        return (x, y, u, loss, lse, dz, dd, dx, dw, db, ops.embed_tokens_backward(dx, self.tokens, self.vocab, scale=2.0)) + \
            tuple(outs) + tuple(step[1:])


def test_a_captured_run_replays():
    announce("token operators captured")
    run = _Run(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = run()
    for replay in range(4):
        run.renew()
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(captured, run())):
            assert torch.equal(a, b), (replay, k)
        torch.cuda.synchronize()


def test_graphs_of_one_stream_replay_on_several():
    """Two graphs captured on one stream have nothing in common: replayed at once, each gives its own results."""
    from gear_amd import ops
    announce("two graphs of token operators at once")
    g = torch.Generator(device="cuda").manual_seed(9)
    runs = []
    for n in (60000, 50000):
        tokens = torch.randint(0, 300, (n,), generator=g, device="cuda")
        dout, w = torch.randn(n, 256, generator=g, device="cuda"), torch.ones(256, device="cuda")
        logits = torch.randn(40, 150000, generator=g, device="cuda")
        runs.append(lambda tokens=tokens, dout=dout, w=w, logits=logits: (
            ops.embed_tokens_backward(dout, tokens, 300),) + ops.layer_norm_backward(dout, dout, w, w) + ops.token_log_probs(logits, top=6)[1:])
    want = [run() for run in runs]
    side, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in runs]
    with torch.cuda.stream(side):
        runs[0]()  # (scratch of this stream is there already)
    torch.cuda.synchronize()
    graphs, captured = [], []
    for run in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.append(run())
        graphs.append(graph)
    for replay in range(6):
        for graph, stream in zip(graphs, others):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, captured):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), replay


def test_streams_and_threads():
    """Calls at once from several threads, each on a stream of its own and two on the same: the results of one alone."""
    announce("token operators on streams and threads")
    runs = [_Run(seed, rows=5000 if seed == 2 else 700) for seed in (2, 3, 4, 5)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got, errors = [None] * 4, []

    def work(k):
        try:
            with torch.cuda.stream(streams[min(k, 2)]):
                for _ in range(5):
                    got[k] = runs[k]()
        except Exception as e:  # pragma: no cover
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def _windows(vocab, step, batch=6, steps=7, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(0, vocab, (batch, steps, step), generator=g, device="cuda")
    mask, done = torch.ones(batch, steps, dtype=torch.uint8, device="cuda"), torch.zeros(batch, steps, dtype=torch.uint8, device="cuda")
    mask[0, :3], mask[1, 5:], done[2, 4] = 0, 0, 1
    return tokens, mask, done


@pytest.mark.parametrize("parameters", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [37, 3000])
def test_model_against_torch(vocab, parameters):
    """The logits are those of the same model with its lookups and norms in torch, and so are the gradients."""
    from gear_amd import sequence
    from gear_amd.sequence import TokenModel
    announce("token model %d %s" % (vocab, parameters))
    torch.manual_seed(0)
    model = TokenModel(vocab, 4, width=64, heads=2, kv_heads=1, dtype=torch.float16).cuda().to(parameters)
    tokens, mask, done = _windows(vocab, 4)
    names = [n for n, _ in model.named_parameters()]

    def grads():
        model.zero_grad()
        logp, entropy = model.log_probs(tokens, mask, done)[:2]
        (-(logp.sum() + 0.1 * entropy.sum()) / 42).backward()
        return logp.detach(), entropy.detach(), [p.grad.float() for p in model.parameters()]

    got = grads()
    assert all(p.grad.dtype == parameters for p in model.parameters())
    kept = {n: getattr(sequence, n) for n in ("embed_tokens", "layer_norm", "token_log_probs")}

    def log_probs(logits, tokens, scale=1.0, top=0):
        l = torch.log_softmax(logits.float() * scale, -1)
        live = tokens >= 0
        return (torch.where(live, l.gather(-1, tokens.clamp(min=0)[..., None])[..., 0], 0.0), torch.where(live, -(l.exp() * l).sum(-1), 0.0))

    def norm(x, w, b, residual=None, eps=1e-5):
        u = x if residual is None else x + residual
        y = torch.nn.functional.layer_norm(u.float(), u.shape[-1:], w.float(), b.float(), eps).to(u.dtype)
        return y if residual is None else (y, u)

    try:
        sequence.embed_tokens = lambda t, table, scale: (torch.nn.functional.embedding(t, table).float() * scale).to(table.dtype)
        sequence.layer_norm, sequence.token_log_probs = norm, log_probs
        want = grads()
    finally:
        for n, f in kept.items():
            setattr(sequence, n, f)
    # two layers of operands of O(1): the roundings of the coarser type, or of attention's f16
    unit = max(torch.finfo(parameters).eps, 2.0 ** -10)
    assert float((got[0] - want[0]).abs().max()) < 32 * unit and float((got[1] - want[1]).abs().max()) < 32 * unit
    for n, a, b in zip(names, got[2], want[2]):
        assert float((a - b).norm()) <= 32 * unit * float(b.norm()) + 1e-6, n


def test_padding_does_not_matter():
    from gear_amd.sequence import TokenModel
    announce("token model: padding")
    torch.manual_seed(1)
    model = TokenModel(50, 3, width=64, heads=2, kv_heads=1).cuda()
    tokens, mask, done = _windows(50, 3)
    outs = model.log_probs(tokens, mask, done, top=4)
    other = torch.where(mask[..., None] == 0, -1, tokens)
    again = model.log_probs(other, mask, done, top=4)
    for a, b in zip(outs, again):
        assert torch.equal(a, b)
    assert float(outs[0].detach()[mask == 0].abs().max()) == 0 and bool((outs[4][mask == 0] == -1).all())
    # a student that is its teacher has little to learn from all of its actions, and padding no part in it
    loss = model.distilled(model, tokens, mask, done, count=50)
    assert float(loss.detach().abs().max()) < 50 * 2.0 ** -22 and float(loss.detach()[mask == 0].abs().max()) == 0


def test_rollouts():
    """Step by step out of caches: the distributions of the whole window."""
    from gear_amd.sequence import Rollouts, TokenModel
    announce("token model: rollouts")
    torch.manual_seed(2)
    model = TokenModel(40, 5, width=64, heads=2, kv_heads=1, dtype=torch.float16).cuda()
    g = torch.Generator(device="cuda").manual_seed(7)
    tokens = torch.randint(0, 40, (9, 6, 5), generator=g, device="cuda")
    ones = torch.ones(9, 6, dtype=torch.uint8, device="cuda")
    with torch.no_grad():
        want = model.log_probs(tokens, ones, ones * 0, top=40)
    rollouts = Rollouts(model, 9, 5 * 6 - 1)
    for t in range(6):
        entropy, value, best = model.step(rollouts, tokens[:, t, :4], tokens[:, t - 1, 4] if t else None, top=40)
        assert float((entropy - want[1][:, t]).abs().max()) < 64 * 2.0 ** -11
        back = torch.zeros(9, 40, device="cuda").scatter(1, best, value)
        whole = torch.zeros(9, 40, device="cuda").scatter(1, want[4][:, t], want[3][:, t])
        assert float((back - whole).abs().max()) < 64 * 2.0 ** -11
    assert rollouts.length.flatten().tolist() == [29] * 9
    with pytest.raises(ValueError, match="caches of 29 tokens hold 29: no room for 5 more"):
        model.step(rollouts, tokens[:, 0, :4], tokens[:, 0, 4])


def test_the_example():
    spec = importlib.util.spec_from_file_location("train_token_model", os.path.join(ROOT, "examples", "train_token_model.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    announce("the example of token models")
    torch.manual_seed(0)
    teacher, student = example.model().cuda(), example.model(width=64, layers=1).cuda()
    batches = example.loader(example.dataset(64, key=os.getpid() + 78), 64)
    before = [p.detach().clone() for p in student.parameters()]
    for losses in (example.clone(teacher, batches, 4), example.distil(student, teacher, batches, 4)):
        assert losses.shape == (4,) and bool(torch.isfinite(losses).all())
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for m in (teacher, student) for p in m.parameters())
    assert all(not torch.equal(a, b) for a, b in zip(before, student.parameters()))
    assert example.act(student, 16).shape == (16, example.SPAN)
