"""Performance cases of the operators at both ends of a sequence model of tokens, and between its blocks.

A case names its `kind` and its sizes:

  embed      tokens -> rows of a table; `train`: with the gradient of the table
  norm       layer norm of rows; `residual`: of their sum with a second input, which is returned as well; `train`: with
             the gradients of the rows, the weight and the bias
  logprobs   logits -> log probabilities of given tokens (`given`), entropies, the `top` best tokens; `train`: with the
             gradient of the logits
  distill    logits and a teacher's best `top` tokens -> the divergence; `train`: with the gradient of the logits

`beside`: rows are every second one of what a projection left (a step's observation and action tokens lie side by side).
With `own` false a pass computes the operator's definition from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-5
PAD = 0.03  # share of the tokens that are padding (-1)


def listed():
    return [
        # the newest two tokens of 64 rollouts: the smallest call
        dict(name="embed_step", kind="embed", N=128, V=1025, W=256, dtype="float16", tokens="bins", train=False),
        # a training batch of 2048 windows of 90 tokens, values in 1024 bins and a separator: a few bins hold most of them
        dict(name="embed_windows", kind="embed", N=2048 * 90, V=1025, W=512, dtype="bfloat16", tokens="bins", train=True),
        # instructions and bins in one vocabulary, trained in 32 bits: few tokens for a large table, some words everywhere
        dict(name="embed_words", kind="embed", N=16 * 1001, V=33025, W=768, dtype="float32", tokens="words", train=True),
        # the norm after a block of one step of 64 rollouts
        dict(name="norm_step", kind="norm", N=192, W=512, dtype="bfloat16", residual=True, beside=False, train=False),
        # 2048 windows of 60 tokens through a narrow model in 32 bits
        dict(name="norm_windows", kind="norm", N=2048 * 60, W=128, dtype="float32", residual=False, beside=False, train=True),
        # 30-step windows of frame patches through a wide model, the sum with the block's output in the same pass
        dict(name="norm_frames", kind="norm", N=32 * 1470, W=2048, dtype="bfloat16", residual=True, beside=False, train=True),
        # a discrete policy with 18 actions, some not allowed: policy gradients with an entropy bonus
        dict(name="actions_windows", kind="logprobs", N=2048 * 90, V=18, dtype="float32", top=0, given=True, masked=True,
             beside=False, train=True),
        # training on tokens of a large vocabulary, odd rows: the largest call
        dict(name="tokens_windows", kind="logprobs", N=16384, V=33025, dtype="bfloat16", top=0, given=True, masked=False,
             beside=False, train=True),
        # the next token of 64 rollouts: few rows of a large vocabulary, the best eight
        dict(name="tokens_step", kind="logprobs", N=64, V=65537, dtype="float16", top=8, given=False, masked=False,
             beside=False, train=False),
        # a teacher's best 32 tokens over a batch
        dict(name="tokens_teacher", kind="logprobs", N=4096, V=33024, dtype="bfloat16", top=32, given=False, masked=False,
             beside=False, train=False),
        # a small batch of 20-step windows in 1024 bins: launches count
        dict(name="distill_small", kind="distill", N=1280, V=1024, dtype="float16", top=8, beside=False, train=True),
        # a batch learnt from the teacher's best 32
        dict(name="distill_windows", kind="distill", N=8191, V=33025, dtype="bfloat16", top=32, beside=False, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "logprobs", "logprobs", "distill"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    train, beside = rng.random() < 0.7, rng.random() < 0.2
    if kind == "embed":
        W = rng.choice([_log(rng, 1, 4096), 8 * _log(rng, 1, 512)])
        N = _log(rng, 1, min(300000, 2048 * 90 * 512 // W))
        return dict(kind=kind, N=N, V=_log(rng, 2, min(70000, 100000000 // W)), W=W, dtype=dtype,
                    tokens=rng.choice(["bins", "words"]), train=train)
    if kind == "norm":
        W = rng.choice([_log(rng, 16, 16384), 8 * _log(rng, 2, 2048)])
        return dict(kind=kind, N=_log(rng, 1, min(300000, 32 * 1470 * 2048 // 2 // W)), W=W, dtype=dtype,
                    residual=rng.random() < 0.5, beside=beside, train=train)
    V = rng.choice([_log(rng, 2, 150000), _log(rng, 2, 2000), 8 * _log(rng, 1, 8192)])
    N = _log(rng, 1, max(1, min(200000, 16384 * 33025 // 4 // V)))
    scale = rng.choice([1.0, 1.0, 0.7])
    if kind == "distill":
        return dict(kind=kind, N=N, V=V, dtype=dtype, scale=scale, top=rng.randint(1, min(V, 64)), beside=beside, train=train)
    top = rng.choice([0, 0, rng.randint(1, min(V, 64)), 1])
    given = top == 0 or rng.random() < 0.5
    return dict(kind=kind, N=N, V=V, dtype=dtype, scale=scale, top=top, given=given, masked=top == 0 and rng.random() < 0.3,
                beside=beside, train=train and given)


# ---- inputs ------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _rows(g, case, width, scale):
    """[N, width] rows; `beside`: every second one of twice as many."""
    n = case["N"]
    return _normal(g, (n, 2, width), DTYPES[case["dtype"]], scale)[:, 1] if case["beside"] else \
        _normal(g, (n, width), DTYPES[case["dtype"]], scale)


def _padding(g, n):
    return torch.rand(n, generator=g, device="cuda") < PAD


def _tokens(g, n, V, kind):
    if kind == "bins":  # values around the middle of their range
        t = (V / 2 + V / 10 * torch.randn(n, generator=g, device="cuda")).round().clamp(0, V - 1).long()
    else:  # the k-th most frequent word once in k, in no order
        t = torch.exp(torch.rand(n, generator=g, device="cuda") * math.log(V)).long().clamp(max=V) - 1
        t = t.clamp(min=0) * 7919 % V
    return torch.where(_padding(g, n), -1, t)


def _drawn(g, logits):
    """A token of each row, by its probabilities."""
    noise = torch.rand(logits.shape, generator=g, device="cuda").clamp_(min=1e-30).log_().neg_().clamp_(min=1e-30).log_()
    return (logits.float() - noise).argmax(-1)


def prepare(case, seed):
    s = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed + 5)
    kind, n, dtype = case["kind"], case["N"], DTYPES[case["dtype"]]
    if kind == "embed":
        s["ids"] = _tokens(g, n, case["V"], case["tokens"])
        s["table"] = _normal(g, (case["V"], case["W"]), dtype, 0.5)
        s["scale"] = math.sqrt(case["W"])
        if case["train"]:
            s["gout"] = _normal(g, (n, case["W"]), dtype)
        return s
    if kind == "norm":
        W = case["W"]
        s["x"] = _rows(g, case, W, 1.5)
        s["r"] = _normal(g, (n, W), dtype) if case["residual"] else None
        s["w"] = (1 + 0.2 * torch.randn(W, generator=g, device="cuda"))
        s["b"] = (0.2 * torch.randn(W, generator=g, device="cuda"))
        if case["train"]:
            s["gy"] = _normal(g, (n, W), dtype)
            s["gsum"] = _normal(g, (n, W), dtype) if case["residual"] else None
        return s
    V = case["V"]
    s["scale"] = case.get("scale", 1.0)
    s["logits"] = _rows(g, case, V, 2.5)
    if kind == "distill":
        # a teacher that agrees in part
        t = s["logits"].float() + 1.5 * torch.randn(n, V, generator=g, device="cuda")
        value, s["best"] = torch.topk(t, case["top"])
        s["teacher"] = value - torch.logsumexp(t, -1, keepdim=True)
        s["best"] = torch.where(_padding(g, n)[:, None], -1, s["best"])
        if case["train"]:
            s["gloss"] = torch.rand(n, generator=g, device="cuda") + 0.5
        return s
    if case["masked"]:  # an action may not be allowed; the first that is drawn is one that is
        hidden = torch.rand(n, V, generator=g, device="cuda") < 0.3
        hidden.scatter_(1, torch.randint(0, V, (n, 1), generator=g, device="cuda"), False)
        s["logits"] = s["logits"].masked_fill(hidden, float("-inf"))
    s["ids"] = None
    if case["given"]:
        s["ids"] = torch.where(_padding(g, n), -1, _drawn(g, s["logits"]))
    if case["train"]:
        s["glogp"], s["gent"] = (torch.randn(2, n, generator=g, device="cuda") * torch.tensor([[1.0], [0.1]], device="cuda")).unbind(0)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------

def _embed(s):
    ids, V = s["ids"], s["V"]
    dtype = DTYPES[s["dtype"]]
    valid = ((ids >= 0) & (ids < V))[:, None]
    out = (torch.where(valid, s["table"].float()[ids.clamp(0, V - 1)], 0.0) * s["scale"]).to(dtype)
    if not s["train"]:
        return out
    # thousands of rows go into some sums: 32 bits would not do for a result in 32
    wide = torch.float64 if dtype == torch.float32 else torch.float32
    sums = torch.zeros(V + 1, s["W"], dtype=wide, device="cuda")
    sums.index_add_(0, torch.where(valid[:, 0], ids, V), s["gout"].to(wide))
    return out, (sums[:V] * s["scale"]).to(dtype)


def _norm(s):
    dtype = DTYPES[s["dtype"]]
    u = s["x"]
    if s["residual"]:
        u = (s["x"].float() + s["r"].float()).to(dtype)
    x = u.float()
    c = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS)
    n = c * rstd
    y = (n * s["w"] + s["b"]).to(dtype)
    outs = (y, u) if s["residual"] else (y,)
    if not s["train"]:
        return outs
    gy = s["gy"].float()
    h = gy * s["w"]
    dx = rstd * (h - h.mean(-1, keepdim=True) - n * (h * n).mean(-1, keepdim=True))
    if s["residual"]:
        dx = dx + s["gsum"].float()
    return outs + (dx.to(dtype), (gy * n).sum(0), gy.sum(0))


def _log_softmax(s):
    z = s["logits"].float() * s["scale"]
    top = z.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(z - top).sum(-1, keepdim=True)) + top
    return z - lse, lse[:, 0]


def _best(logits, k):
    """The k largest of a row and where they are, the lower index first among equals."""
    bits = (logits.float() + 0.0).contiguous().view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
    key += torch.arange(logits.shape[1] - 1, -1, -1, device="cuda")
    return logits.shape[1] - 1 - (torch.topk(key, k).values & 0xFFFFFFFF)


def _logprobs(s):
    logp, lse = _log_softmax(s)
    p = torch.exp(logp)
    logp_finite = torch.where(p > 0, logp, 0.0)  # (what is not allowed has no part in the entropy)
    entropy = -(p * logp_finite).sum(-1)
    outs = []
    valid = None
    if s["given"]:
        ids = s["ids"]
        valid = (ids >= 0) & (ids < s["V"])
        at = ids.clamp(0, s["V"] - 1)[:, None]
        outs.append(torch.where(valid, logp.gather(1, at)[:, 0], 0.0))
        entropy, lse = torch.where(valid, entropy, 0.0), torch.where(valid, lse, 0.0)
    outs += [entropy, lse]
    if s["top"]:
        best = _best(s["logits"], s["top"])
        value = logp.gather(1, best)
        if valid is not None:
            value, best = torch.where(valid[:, None], value, float("-inf")), torch.where(valid[:, None], best, -1)
        outs += [value, best]
    if s["train"]:
        gl, ge = torch.where(valid, s["glogp"], 0.0)[:, None], torch.where(valid, s["gent"], 0.0)[:, None]
        d = p * (-gl - ge * (logp_finite + entropy[:, None]))
        d.scatter_add_(1, at, gl)
        outs.append((d * s["scale"]).to(DTYPES[s["dtype"]]))
    return tuple(outs)


def _distill(s):
    logp, lse = _log_softmax(s)
    best, there = s["best"], s["best"] >= 0
    some = there.any(-1)
    t = torch.where(there, s["teacher"], float("-inf"))
    e = torch.exp(t - t.amax(-1, keepdim=True).clamp(min=-3e38))
    total = e.sum(-1, keepdim=True)
    q = e / torch.where(total > 0, total, 1.0)
    at = best.clamp(min=0)
    loss = (q * (torch.log(torch.where(q > 0, q, 1.0)) - torch.where(q > 0, logp.gather(1, at), 0.0))).sum(-1)
    outs = (loss, torch.where(some, lse, 0.0))
    if not s["train"]:
        return outs
    g = torch.where(some, s["gloss"], 0.0)[:, None]
    d = torch.exp(logp) * g
    d.scatter_add_(1, at, -q * g)
    return outs + ((d * s["scale"]).to(DTYPES[s["dtype"]]),)


def run(s):
    if own:
        return _run_own(s)
    return {"embed": _embed, "norm": _norm, "logprobs": _logprobs, "distill": _distill}[s["kind"]](s)


# ---- the framework's operators -----------------------------------------------------------------------------

def _run_own(s):
    from gear_amd import ops
    kind = s["kind"]
    if kind == "embed":
        out = ops.embed_tokens(s["ids"], s["table"], scale=s["scale"])
        if not s["train"]:
            return out
        return out, ops.embed_tokens_backward(s["gout"], s["ids"], s["V"], scale=s["scale"])
    if kind == "norm":
        y = ops.layer_norm(s["x"], s["w"], s["b"], residual=s["r"], eps=EPS)
        outs, u = (y, y[1]) if s["residual"] else ((y,), s["x"])
        if not s["train"]:
            return outs
        return outs + ops.layer_norm_backward(s["gy"], u, s["w"], s["b"], dsum=s["gsum"], eps=EPS)
    if kind == "distill":
        loss, lse = ops.distill(s["logits"], s["best"], s["teacher"], scale=s["scale"])
        if not s["train"]:
            return loss, lse
        return loss, lse, ops.distill_backward(s["gloss"], s["logits"], s["best"], s["teacher"], lse, scale=s["scale"])
    logp, entropy, lse, value, best = ops.token_log_probs(s["logits"], s["ids"], scale=s["scale"], top=s["top"])
    outs = tuple(x for x in (logp, entropy, lse, value, best) if x is not None)
    if not s["train"]:
        return outs
    return outs + (ops.token_log_probs_backward(s["glogp"], s["gent"], s["logits"], s["ids"], lse, entropy, scale=s["scale"]),)


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    kind, n, train = case["kind"], case["N"], case["train"]
    size = 4 if case["dtype"] == "float32" else 2
    if kind == "embed":
        V, W = case["V"], case["W"]
        used = min(n, V) * W
        return {"bytes": size * (used + n * W + train * (n * W + V * W)) + 8 * n, "flops": n * W * (1 + train)}
    if kind == "norm":
        passes = (2 + 2 * case["residual"]) + train * (3 + case["residual"])
        return {"bytes": size * passes * n * case["W"] + 16 * case["W"], "flops": n * case["W"] * (8 + 14 * train)}
    V = case["V"]
    read = n * V * size * (1 - PAD * (kind == "distill" or case["given"]))
    each = 12 * case["top"] + 8
    if kind == "distill":
        return {"bytes": int(read * (1 + train) + train * n * V * size) + n * (each * (1 + train) + 8 * train), "flops": n * V * (6 + 5 * train)}
    each += 12 * case["given"]
    return {"bytes": int(read * (1 + train) + train * n * V * size) + n * each * (1 + train), "flops": n * V * (8 + 9 * train)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def _exact_embed(s):
    V, W = s["V"], s["W"]
    inside = (s["ids"] >= 0) & (s["ids"] < V)
    out = torch.zeros(s["N"], W, dtype=torch.float64, device="cuda")
    out[inside] = s["table"].double()[s["ids"][inside]] * s["scale"]
    if not s["train"]:
        return out
    # the rows of a token stand together in token order: differences of running sums
    order = torch.argsort(s["ids"][inside])
    ids = s["ids"][inside][order]
    ends = torch.searchsorted(ids, torch.arange(-1, V, device="cuda"), right=True)
    grad = torch.empty(V, W, dtype=torch.float64, device="cuda")
    for a in range(0, W, 256):
        rows = s["gout"][:, a:a + 256].double()[inside][order]
        total = torch.nn.functional.pad(rows.cumsum(0), (0, 0, 1, 0))[ends]
        grad[:, a:a + 256] = (total[1:] - total[:-1]) * s["scale"]
    return out, grad


def _exact_norm(s):
    def f(u, w, b):
        centre = u - u.sum(-1, keepdim=True) / s["W"]
        return centre / torch.sqrt((centre * centre).sum(-1, keepdim=True) / s["W"] + EPS) * w + b

    # (the norm is of the sum as it is stored)
    u = (s["x"].double() + s["r"].double()).to(DTYPES[s["dtype"]]).double() if s["residual"] else s["x"].double()
    w, b = s["w"].double().requires_grad_(), s["b"].double().requires_grad_()
    ys, dx, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for a in range(0, s["N"], 16384):
        part = u[a:a + 16384].clone().requires_grad_()
        y = f(part, w, b)
        ys.append(y.detach())
        if s["train"]:
            gx, gw, gb = torch.autograd.grad(y, (part, w, b), s["gy"][a:a + 16384].double())
            dx.append(gx + s["gsum"][a:a + 16384].double() if s["residual"] else gx)
            dw, db = dw + gw, db + gb
    outs = (torch.cat(ys), u) if s["residual"] else (torch.cat(ys),)
    return outs + (torch.cat(dx), dw.detach(), db.detach()) if s["train"] else outs


def _chunks(s):
    rows = max(1, int(5e7) // s["V"])
    return [slice(a, min(a + rows, s["N"])) for a in range(0, s["N"], rows)]


def _exact_logprobs(s):
    """By probabilities: sums and quotients of exponentials, gradients by autograd."""
    parts = []
    for c in _chunks(s):
        x = s["logits"][c].double()
        seen = torch.isfinite(x)
        z = torch.where(seen, x, 0.0).requires_grad_()
        shift = torch.where(seen, x, -1e300).amax(-1, keepdim=True) * s["scale"]
        e = torch.where(seen, torch.exp(z * s["scale"] - shift), 0.0)
        norm = e.sum(-1, keepdim=True)
        p = e / norm
        entropy = -torch.where(p > 0, p * torch.log(torch.where(p > 0, p, 1.0)), 0.0).sum(-1)
        lse = (torch.log(norm) + shift)[:, 0]
        row, outs, alive = torch.arange(len(x), device="cuda"), [], torch.ones(len(x), dtype=torch.float64, device="cuda")
        if s["given"]:
            ids = s["ids"][c]
            alive = (ids >= 0).double()
            logp = (z[row, ids.clamp(min=0)] * s["scale"] - lse) * alive
            outs.append(logp.detach())
        outs += [(entropy * alive).detach(), (lse * alive).detach()]
        if s["top"]:
            best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["top"]]
            value = torch.log(p.detach().gather(1, best))
            outs += [torch.where(alive[:, None] > 0, value, float("-inf")), torch.where(alive[:, None] > 0, best, -1)]
        if s["train"]:
            loss = (s["glogp"][c].double() * logp + s["gent"][c].double() * entropy * alive).sum()
            outs.append(torch.autograd.grad(loss, z)[0])
        parts.append(outs)
    return tuple(torch.cat(x) for x in zip(*parts))


def _exact_distill(s):
    parts = []
    for c in _chunks(s):
        z = s["logits"][c].double().requires_grad_()
        there = s["best"][c] >= 0
        lse = torch.logsumexp(z * s["scale"], -1)
        weight = torch.where(there, torch.exp(s["teacher"][c].double()), 0.0)
        total = weight.sum(-1, keepdim=True)
        q = weight / torch.where(total > 0, total, 1.0)
        mine = z.gather(1, s["best"][c].clamp(min=0)) * s["scale"] - lse[:, None]
        loss = (torch.special.xlogy(q, q) - q * mine).sum(-1)
        outs = [loss.detach(), torch.where(total[:, 0] > 0, lse.detach(), 0.0)]
        if s["train"]:
            outs.append(torch.autograd.grad((loss * s["gloss"][c].double()).sum(), z)[0])
        parts.append(outs)
    return tuple(torch.cat(x) for x in zip(*parts))


def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "norm": _exact_norm, "logprobs": _exact_logprobs, "distill": _exact_distill}[case["kind"]](s)
