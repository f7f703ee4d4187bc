"""The operators of token models where offsets pass 32 bits, where a token is most of a batch, and where rows are in parts, on
several streams and captured."""
import threading

import pytest

from conftest import announce
from sequence_reference import worst
from tokens_reference import TYPES, LayerNorm, LogProbs, embed_backward, rounded, teacher

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BORDER = 1 << 31


def _some(rows, width):
    """The first and last rows, and those around the element of number 2^31."""
    at = BORDER // width
    return torch.tensor(sorted({r for r in (0, 1, at - 1, at, at + 1, rows - 2, rows - 1) if 0 <= r < rows}), device="cuda")


def _many(rows, width, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    assert rows * width > BORDER
    return torch.randn(rows, width, generator=g, device="cuda", dtype=torch.bfloat16), g


def _check_logits(x, g, pick):
    """x [rows, vocab] as a whole through the operators, the picked rows against 64 bits."""
    from gear_amd import ops
    rows, vocab = x.shape
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    dl, de = torch.rand(2, rows, generator=g, device="cuda")
    logp, entropy, lse, value, best = ops.token_log_probs(x, tokens, top=4)
    ref = LogProbs(x[pick], 1.0)
    at = tokens[pick][:, None]
    assert worst(logp[pick], ref.logp.gather(1, at)[:, 0], ref.logp_bound(ref.logp.gather(1, at)[:, 0], ref.d.gather(1, at)[:, 0])) <= 1
    assert worst(entropy[pick], ref.entropy, ref.entropy_bound) <= 1 and worst(lse[pick], ref.lse, ref.lse_bound) <= 1
    logs = ref.logp.gather(1, best[pick])
    assert worst(value[pick], logs, ref.s_error[:, None] + 2.0 ** -24 * (4 * ref.d.gather(1, best[pick]).abs() + 2 * logs.abs() + 4)) <= 1
    assert torch.equal(x[pick].gather(1, best[pick]), torch.topk(x[pick].float(), 4).values.to(x.dtype))
    got = ops.token_log_probs_backward(dl, de, x, tokens, lse, entropy)[pick]
    a, b, h = dl[pick].double()[:, None], de[pick].double()[:, None], ref.entropy[:, None]
    one = torch.zeros_like(ref.p).scatter_(1, at, 1.0)
    want, bound = ref.gradient(-a - b * h, -b, a * one, x.dtype, ref.lse, a + b * (1 + h + ref.entropy_bound[:, None] * 2 ** 20))
    assert worst(got, want, bound) <= 1
    del got
    t = value.clone()
    loss, lse = ops.distill(x, best, t)
    got = ops.distill_backward(dl, x, best, t, lse)[pick]
    q, q_error, _ = teacher(best[pick], t[pick], vocab)
    weight, error = (torch.zeros_like(ref.p).scatter_(1, best[pick], v) for v in (q, q_error))
    want, bound = ref.gradient(a, torch.zeros_like(a), -a * weight, x.dtype, ref.lse, a)
    assert worst(got, want, bound + a * (error + 2.0 ** -24 * 66 * weight)) <= 1
    each = torch.log(q) - logs
    bound = (q_error * (each.abs() + 1) + q * (ref.s_error[:, None] + 2.0 ** -24 * (4 * ref.d.gather(1, best[pick]).abs() + 80 * each.abs() + 80))).sum(-1)
    assert worst(loss[pick], (q * each).sum(-1), bound) <= 1


@pytest.mark.parametrize("rows,vocab", [(2200003, 1001), (65551, 33025)])
def test_more_than_2_31_logits(rows, vocab):
    announce("logits %d x %d" % (rows, vocab))
    x, g = _many(rows, vocab, 1)
    _check_logits(x, g, _some(rows, vocab))


@pytest.mark.parametrize("vocab", [1001, 5000])
def test_rows_of_logits_far_apart(vocab):
    """Three rows, each more than 2^30 elements from the next."""
    announce("logits far apart %d" % vocab)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(3, (1 << 30) + 12345, device="cuda", dtype=torch.bfloat16)[:, 7:7 + vocab]
    x.copy_(torch.randn(3, vocab, generator=g, device="cuda"))
    _check_logits(x, g, torch.arange(3, device="cuda"))


def test_more_than_2_31_elements_of_tables():
    from gear_amd import ops
    announce("embed: a table of more than 2^31 elements")
    table, g = _many(2200003, 1001, 3)
    pick = _some(*table.shape)
    tokens = torch.cat([pick, torch.randint(0, len(table), (500,), generator=g, device="cuda"), pick[-1:]])
    out = ops.embed_tokens(tokens, table)
    assert torch.equal(out, table[tokens])
    del table
    grad = ops.embed_tokens_backward(out, tokens, 2200003)
    named = torch.unique(tokens)
    ref, bound = embed_backward(out, torch.searchsorted(named, tokens), len(named), 1.0)
    assert worst(grad[named], ref, bound) <= 1
    assert int(grad.any(1).sum()) == len(named)


def test_more_than_2_31_elements_of_rows():
    from gear_amd import ops
    announce("embed: rows of more than 2^31 elements")
    dout, g = _many(2200003, 1001, 4)
    pick = _some(*dout.shape)
    tokens = torch.randint(0, 50, (len(dout),), generator=g, device="cuda")
    tokens[pick] = 50 + torch.arange(len(pick), device="cuda")
    grad = ops.embed_tokens_backward(dout, tokens, 60, scale=2.0)
    assert torch.equal(grad[50:50 + len(pick)], dout[pick] * 2) and float(grad[50 + len(pick):].abs().sum()) == 0
    # 44 000 numbers of size 0.8 each: 256 of a chunk one after the other, then 170 chunks by 16 waves, in 32 bits; one rounding
    part = torch.zeros(50, 1001, dtype=torch.float64, device="cuda")
    for rows, names in zip(dout.split(200000), tokens.split(200000)):
        part.index_add_(0, names.clamp(max=49), torch.where((names < 50)[:, None], rows.double(), 0.0))
    assert float((grad[:50].double() - 2 * part).abs().max()) <= 2.0 ** -8 * float(2 * part.abs().max()) + 2.0 ** -24 * 400 * 2 * 50000
    del grad
    table = torch.randn(50, 1001, generator=g, device="cuda").bfloat16()
    out = ops.embed_tokens(tokens, table)
    assert torch.equal(out[:pick[2]][::1000], torch.where((tokens < 50)[:, None], table[tokens.clamp(max=49)], 0.0)[:pick[2]][::1000])
    assert float(out[pick].abs().sum()) == 0 and torch.equal(out[-5:-2], table[tokens[-5:-2]])


def test_more_than_2_31_elements_of_norms():
    from gear_amd import ops
    announce("layer_norm: more than 2^31 elements")
    x, g = _many(2200003, 1001, 5)
    r, dsum = x.flip(0), x.roll(1, 0)
    pick = _some(*x.shape)
    w, b = torch.rand(2, 1001, generator=g, device="cuda")
    y, u = ops.layer_norm(x, w, b, residual=r)
    total = x[pick].double() + r[pick].double()
    assert worst(u[pick], total, rounded(total, x.dtype) + 2.0 ** -24 * total.abs()) <= 1
    del r
    dx, dw, db = ops.layer_norm_backward(x, u, w, b, dsum=dsum)
    ref = LayerNorm(u[pick], w, b, 1e-5, x[pick], dsum[pick])
    assert worst(y[pick], ref.y, ref.y_bound) <= 1 and worst(dx[pick], ref.dx, ref.dx_bound) <= 1
    assert worst(db, sum(rows.double().sum(0) for rows in x.split(200000)), 2.0 ** -24 * (len(x) + 64) * x.float().abs().mean(0).double() * len(x)) <= 1


# 188, 2300 and 1170 chunks of one token, in several tiles of 256 (32 bits) or 512 columns
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,width", [(3000, 1, 1100), (37000, 1, 1030), (150000, 2, 600), (3000, 3, 2049)])
def test_long_runs_in_tiles(n, vocab, width, dtype):
    from gear_amd import ops
    announce("embed: long runs %s n=%d vocab=%d width=%d" % (dtype, n, vocab, width))
    g = torch.Generator(device="cuda").manual_seed(n + width)
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    dout = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    grad = ops.embed_tokens_backward(dout, tokens, vocab, scale=0.5)
    ref, bound = embed_backward(dout, tokens, vocab, 0.5)
    assert worst(grad, ref, bound) <= 1
    assert torch.equal(grad, ops.embed_tokens_backward(dout, tokens, vocab, scale=0.5))


class _Parts:
    """Rows in parts that are joined: log probabilities with the best tokens, distillation from them, and the gradients."""

    def __init__(self, seed, rows, vocab, dtype):
        from gear_amd import _cabi
        lib = _cabi.load()
        assert lib.gear_hip_distill_workspace_bytes(rows, vocab) > 0 and lib.gear_hip_token_log_probs_workspace_bytes(rows, vocab, 5) > 0
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.x = torch.empty(rows, vocab, device="cuda", dtype=dtype)
        self.tokens = torch.empty(rows, device="cuda", dtype=torch.int64)
        self.dl, self.de = torch.randn(2, rows, generator=self.g, device="cuda")
        self.renew()

    def renew(self):
        self.x.copy_(torch.randn(self.x.shape, generator=self.g, device="cuda"))
        self.tokens.copy_(torch.randint(-1, self.x.shape[1], self.tokens.shape, generator=self.g, device="cuda"))

    def __call__(self):
        from gear_amd import ops
        outs = ops.token_log_probs(self.x, self.tokens, top=5)
        loss, lse = ops.distill(self.x, outs[4], outs[3])
        return outs + (loss, lse, ops.token_log_probs_backward(self.dl, self.de, self.x, self.tokens, outs[2], outs[1]),
                       ops.distill_backward(self.dl, self.x, outs[4], outs[3], lse))


SPLIT = [(3, 60001, torch.float32), (300, 40003, torch.bfloat16), (5, 150001, torch.float16)]


def test_parts_captured():
    announce("rows in parts captured")
    runs = [_Parts(k, *shape) for k, shape in enumerate(SPLIT)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for run in runs:
            run()
    torch.cuda.synchronize()
    graphs, captured = [], []
    for run in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.append(run())
        graphs.append(graph)
    others = [torch.cuda.Stream() for _ in runs]
    for replay in range(4):
        for run in runs:
            run.renew()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, others):  # all at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for run, outs in zip(runs, captured):
            for k, (a, b) in enumerate(zip(outs, run())):
                assert torch.equal(a, b), (replay, k)
        torch.cuda.synchronize()


def test_parts_on_streams_and_threads():
    """Calls at once from several threads, two of them on one stream: the results of one alone."""
    announce("rows in parts on streams and threads")
    runs = [_Parts(k, *shape) for k, shape in enumerate(SPLIT + SPLIT[:1])]
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
