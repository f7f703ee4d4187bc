"""Performance cases of the operators that take a batch of trajectory windows into a sequence model.

A case names its `kind` and its sizes:

  ranges     the loader's masks and a `done` column -> the range of keys that each token sees, and positions
  norm       per-head norms of queries and keys with the position rotation; `train`: with the gradients;
             `append`: the keys and values go to a cache, as a rollout does
  attention  attention over ranges of keys; `train`: with the gradients of queries, keys and values
  step       the same for the newest tokens of many rollouts, over their caches

With `own` false a pass computes the operator's definition from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6
BASE = 10000.0


def listed():
    return [
        # a batch of 30-step frame windows, three tokens a step (return, frame, action); episodes end
        # inside some windows, others are padded at the head
        dict(name="ranges_windows", kind="ranges", B=2048, S=30, tokens=3, rows=0, cols=0, mode="causal", prefix=0),
        # whole trajectories as patches of frames: a step sees its own patches, the first steps are a prompt
        dict(name="ranges_frames", kind="ranges", B=8, S=1000, tokens=49, rows=7, cols=7, mode="step", prefix=4),
        # one step of 64 rollouts: the three new tokens go into the caches (the smallest call)
        dict(name="norm_append", kind="norm", B=64, T=3, Hq=8, Hk=8, D=64, sections="32", dtype="float16",
             train=False, append=300),
        # 20-step windows of a locomotion table, trained in 32 bits
        dict(name="norm_windows", kind="norm", B=1024, T=60, Hq=8, Hk=8, D=32, sections="16", dtype="float32",
             train=True, append=0),
        # patches of 30-step frame windows: positions with three axes, shared key heads
        dict(name="norm_frames", kind="norm", B=64, T=1470, Hq=16, Hk=4, D=128, sections="24,20,20",
             dtype="bfloat16", train=True, append=0),
        # a small batch of 20-step windows: launches count
        dict(name="attention_small", kind="attention", B=64, T=60, S=60, Hq=4, Hk=4, D=32, dtype="float16",
             tokens=3, mode="causal", prefix=0, done=0.001, cap=0.0, slopes=False, train=True),
        # the training batch of 2048 30-step windows
        dict(name="attention_windows", kind="attention", B=2048, T=90, S=90, Hq=8, Hk=8, D=64, dtype="bfloat16",
             tokens=3, mode="causal", prefix=0, done=0.001, cap=0.0, slopes=False, train=True),
        # windows of frame patches, scores capped, key heads shared by four
        dict(name="attention_frames", kind="attention", B=32, T=1470, S=1470, Hq=16, Hk=4, D=128, dtype="bfloat16",
             tokens=49, mode="step", prefix=0, done=0.001, cap=30.0, slopes=False, train=True),
        # long trajectories packed one after the other, a bias by distance: the largest call
        dict(name="attention_packed", kind="attention", B=2, T=8193, S=8193, Hq=16, Hk=8, D=128, dtype="bfloat16",
             tokens=3, mode="causal", prefix=0, done=0.0007, cap=0.0, slopes=True, train=True),
        # scoring the last tokens of long trajectories after a prompt that sees itself: ragged sizes
        dict(name="attention_score", kind="attention", B=5, T=1001, S=2997, Hq=12, Hk=4, D=80, dtype="float16",
             tokens=3, mode="causal", prefix=100, done=0.0, cap=50.0, slopes=False, train=False),
        # the next step of 256 rollouts of up to 1000 steps
        dict(name="step_rollouts", kind="step", B=256, T=3, L=3000, Hq=8, Hk=8, D=64, dtype="bfloat16", cap=0.0,
             slopes=False),
        # one token each of a few very long rollouts, eight heads to a key head
        dict(name="step_long", kind="step", B=3, T=1, L=131071, Hq=16, Hk=2, D=128, dtype="bfloat16", cap=0.0,
             slopes=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hk = rng.choice([1, 2, 3, 4, 8])
    return hk * rng.choice([1, 1, 2, 4]), hk


def draw(rng):
    kind = rng.choice(["ranges", "norm", "attention", "attention", "step"])
    if kind == "ranges":
        rows, cols = rng.choice([(0, 0), (0, 0), (rng.randint(2, 8), rng.randint(2, 8))])
        tokens = rows * cols if rows else rng.randint(1, 4)
        S = _log(rng, 1, 2000)
        return dict(kind=kind, B=_log(rng, 1, max(1, min(4096, 400000 // (S * tokens)))), S=S, tokens=tokens, rows=rows,
                    cols=cols, mode=rng.choice(["causal", "step", "document"]), prefix=rng.choice([0, 0, rng.randint(1, 20)]))
    Hq, Hk = _heads(rng)
    D = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128])
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "norm":
        append = rng.choice([0, 0, rng.randint(10, 500)])
        T = rng.randint(1, 4) if append else _log(rng, 1, 2000)
        B = _log(rng, 1, min(2048, 64 * 1470 * 20 * 128 // (T * (Hq + Hk) * D)))
        if append:
            B = max(1, min(B, 200000000 // (append * Hk * D)))
        half = D // 2
        cut = sorted(rng.randint(0, half) for _ in range(2))
        sections = rng.choice([str(half), "%d,%d,%d" % (cut[0], cut[1] - cut[0], half - cut[1]), str(max(1, half // 2))])
        return dict(kind=kind, B=B, T=T, Hq=Hq, Hk=Hk, D=D, sections=sections, append=append, train=not append,
                    dtype=rng.choice([dtype, dtype, "float32"]))
    cap, slopes = rng.choice([0.0, 0.0, 20.0, 50.0]), rng.random() < 0.3
    if kind == "attention":
        tokens = rng.choice([1, 2, 3, 16, 49])
        most = 60000000000 // (Hq * D)  # pairs of tokens: half of the largest listed case's, where all are visible
        S = _log(rng, 1, min(8192, math.isqrt(most)) // tokens) * tokens
        train = rng.random() < 0.7
        T = S if train or rng.random() < 0.5 else _log(rng, 1, S)
        B = _log(rng, 1, max(1, min(2048, most // (T * S), 2048 * 90 * 8 * 64 // (S * Hq * D))))
        return dict(kind=kind, B=B, T=T, S=S, Hq=Hq, Hk=Hk, D=D, dtype=dtype, tokens=tokens,
                    mode=rng.choice(["causal", "causal", "step", "document"]), prefix=rng.choice([0, 0, rng.randint(1, 100)]),
                    done=rng.choice([0.0, 0.001, 0.02]), cap=cap, slopes=slopes, train=train)
    L = _log(rng, 1, 131071)
    T = rng.randint(1, 4)
    B = _log(rng, 1, max(1, min(1024, 3 * 131071 * 2 * 128 // (L * Hk * D))))
    return dict(kind=kind, B=B, T=min(T, L), L=L, Hq=Hq, Hk=Hk, D=D, dtype=dtype, cap=cap, slopes=slopes)


# ---- inputs ------------------------------------------------------------------------------------------------

def _steps(case, seed, device):
    """mask and done of a batch of windows: half of them full, the others with padding at the head or the
    tail, one in a hundred empty."""
    g = torch.Generator(device=device).manual_seed(seed)
    B = case["B"]
    S = case["S"] // case["tokens"] if case["kind"] == "attention" else case["S"]
    u = torch.rand(B, 3, generator=g, device=device)
    length = torch.where(u[:, 0] < 0.5, torch.full((B,), S, device=device), 1 + (u[:, 1] * S).long().clamp(max=S - 1))
    length = torch.where(u[:, 0] > 0.99, torch.zeros_like(length), length)
    at = torch.arange(S, device=device)
    head = u[:, 2:] < 0.7
    mask = torch.where(head, at >= S - length[:, None], at < length[:, None]).to(torch.uint8)
    done = (torch.rand(B, S, generator=g, device=device) < case.get("done", 0.005)).to(torch.uint8)
    return mask, done


def _sections(case):
    return [int(v) for v in case["sections"].split(",")]


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _slopes(case):
    n = case["Hq"]
    if not case["slopes"]:
        return None
    return torch.exp2(-8.0 * torch.arange(1, n + 1, device="cuda", dtype=torch.float32) / n)


def prepare(case, seed):
    s = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed + 7)
    kind, B = case["kind"], case["B"]
    if kind == "ranges":
        s["mask"], s["done"] = _steps(case, seed, "cuda")
        return s
    dtype, Hq, Hk, D = DTYPES[case["dtype"]], case["Hq"], case["Hk"], case["D"]
    if kind == "norm":
        T, sections = case["T"], _sections(case)
        # queries and keys come out of one projection, side by side with the values
        qkv = _normal(g, (B, T, Hq + 2 * Hk, D), dtype, 1.5)
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
        s["wq"], s["wk"] = (1 + 0.2 * torch.randn(2, D, generator=g, device="cuda")).unbind(0)
        s["freqs"] = torch.cat([BASE ** (-torch.arange(n, dtype=torch.float64, device="cuda") / max(n, 1)) for n in sections])
        s["pos"] = torch.randint(0, 1000, (B, T, len(sections)), generator=g, device="cuda", dtype=torch.int32)
        if case["append"]:
            L = case["append"]
            s["k_cache"], s["v_cache"] = _normal(g, (B, L, Hk, D), dtype), _normal(g, (B, L, Hk, D), dtype)
            at = torch.randint(0, max(1, L - T + 1), (B, 1), generator=g, device="cuda")
            s["slots"] = (at + torch.arange(T, device="cuda")).to(torch.int32)
        if case["train"]:
            s["gq"], s["gk"] = _normal(g, (B, T, Hq, D), dtype), _normal(g, (B, T, Hk, D), dtype)
        return s
    T, S = case["T"], case["S"] if kind == "attention" else case["L"]
    s["slopes"] = _slopes(case)
    s["q"] = _normal(g, (B, T, Hq, D), dtype, 1.2)
    s["k"] = _normal(g, (B, S, Hk, D), dtype, 1.2)
    if kind == "attention":
        # the keys were normed and rotated, the values are still beside them in the projection
        s["v"] = _normal(g, (B, S, 2, Hk, D), dtype)[:, :, 1]
        mask, done = _steps(case, seed, "cuda")
        lo, hi, _ = _ranges(mask, done, case["tokens"], case["mode"], case["prefix"], None)
        s["lo"], s["hi"] = lo[:, S - T:].contiguous(), hi[:, S - T:].contiguous()
        if case["train"]:
            s["gout"] = _normal(g, (B, T, Hq, D), dtype)
    else:  # caches, filled to a length of their own, each new token sees the ones before it
        s["v"] = _normal(g, (B, S, Hk, D), dtype)
        u = torch.rand(B, 2, generator=g, device="cuda")
        length = T + (u[:, 0] * (S - T + 1)).long().clamp(max=S - T)
        first = torch.where(u[:, 1] < 0.7, torch.zeros_like(length), (u[:, 1] - 0.7) * length)
        s["hi"] = (length[:, None] - T + 1 + torch.arange(T, device="cuda")).to(torch.int32)
        s["lo"] = torch.minimum(first.to(torch.int32)[:, None], s["hi"] - 1).contiguous()
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------

def _ranges(mask, done, n, mode, prefix, grid):
    B, S = mask.shape
    dev = mask.device
    at = torch.arange(S, device=dev).expand(B, S)
    valid, ends = mask != 0, done != 0
    before = torch.nn.functional.pad(valid & ~ends, (1, 0))[:, :S]
    after = torch.nn.functional.pad(valid, (0, 1))[:, 1:]
    s0 = torch.cummax(torch.where(valid & ~before, at, -1), 1).values
    last = valid & (ends | ~after)
    s1 = torch.cummin(torch.where(last, at, S).flip(1), 1).values.flip(1) + 1
    u = torch.arange(n, device=dev)
    i = at[:, :, None] * n + u
    if mode == "causal":
        hi = i + 1
    elif mode == "step":
        hi = ((at + 1) * n)[:, :, None].expand(B, S, n)
    else:
        hi = (s1 * n)[:, :, None].expand(B, S, n)
    if prefix:
        hi = torch.maximum(hi, (torch.minimum(s0 + prefix, s1) * n)[:, :, None])
    ok = valid[:, :, None]
    lo = torch.where(ok, (s0 * n)[:, :, None].expand(B, S, n), 0)
    hi = torch.where(ok, hi, 0)
    time = torch.where(valid, at - s0, 0)[:, :, None].expand(B, S, n)
    if grid is None:
        pos = time[..., None]
    else:
        pos = torch.stack([time, torch.where(ok, u // grid[1], 0), torch.where(ok, u % grid[1], 0)], -1)
    return (lo.reshape(B, S * n).int(), hi.reshape(B, S * n).int(), pos.reshape(B, S * n, -1).int())


def _rotation(s):
    """cos and sin of a token's angles, [B, T, 1, D/2].  A position times a frequency is taken as whole
    turns in 64 bits: 32 would leave a thousandth of a radian of a late position."""
    sections = _sections(s)
    pos = torch.cat([s["pos"][..., a:a + 1].expand(-1, -1, n) for a, n in enumerate(sections)], -1)
    turn = torch.frac(pos.double() * s["freqs"] / (2 * math.pi)).float() * (2 * math.pi)
    turn = torch.nn.functional.pad(turn, (0, s["D"] // 2 - turn.shape[-1]))[:, :, None]
    return torch.cos(turn), torch.sin(turn)


def _turn(x, c, s):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _norm_rotate(x, w, c, s):
    x = x.float()
    return _turn(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w, c, s)


def _norm_rotate_grad(gy, x, w, c, s):
    x, g = x.float(), _turn(gy.float(), c, -s)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n, h = x * r, g * w
    return r * (h - n * (h * n).mean(-1, keepdim=True)), (g * n).sum((0, 1, 2))


def _scores(s, q, k, place):
    """Scores [B, Hk, G, T, S] before the mask, what the cap's gradient needs, and the mask."""
    B, T, Hq, D = q.shape
    S, Hk = k.shape[1], k.shape[2]
    x = torch.matmul(_grouped(q, Hk), k.float().permute(0, 2, 3, 1)).view(B, Hk, Hq // Hk, T, S) * D ** -0.5
    slope = None
    if s["cap"]:
        t = torch.tanh(x / s["cap"])
        x, slope = t * s["cap"], 1 - t * t
    at = torch.arange(S, device=q.device)
    if s["slopes"] is not None:
        x = x - s["slopes"].view(Hk, -1, 1, 1) * (place[:, None, None, :, None] - at).abs()
    seen = ((at >= s["lo"][..., None]) & (at < s["hi"][..., None]))[:, None, None]
    return x.masked_fill(~seen, float("-inf")), slope


def _grouped(q, Hk):
    """[B, T, Hq, D] -> [B, Hk, G * T, D] in 32 bits"""
    B, T, Hq, D = q.shape
    return q.float().view(B, T, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)


def _ungrouped(x, T):
    """[B, Hk, G * T, D] -> [B, T, Hq, D]"""
    B, Hk, _, D = x.shape
    return x.view(B, Hk, -1, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, -1, D)


def _attend(s, place):
    q, k, v = s["q"], s["k"], s["v"]
    B, T, Hq, D = q.shape
    Hk, S = k.shape[2], k.shape[1]
    x, slope = _scores(s, q, k, place)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(x - top)
    del x
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    lse = (torch.log(total) + top)[..., 0].view(B, Hq, T)
    lse = torch.where(total[..., 0].view(B, Hq, T) == 0, float("-inf"), lse)
    p = p.view(B, Hk, -1, S)
    return torch.matmul(p, v.float().transpose(1, 2)), lse, p, slope


def _attend_grad(s, out, p, slope):
    q, k, v, T = s["q"], s["k"], s["v"], s["T"]
    Hk, D = k.shape[2], q.shape[3]
    g = _grouped(s["gout"], Hk)
    dv = torch.matmul(p.transpose(2, 3), g)
    d = torch.matmul(g, v.float().permute(0, 2, 3, 1)) - (g * out).sum(-1, keepdim=True)
    d = d * p
    if slope is not None:
        d = d * slope.view(d.shape)
    d = d * D ** -0.5
    dq = torch.matmul(d, k.float().transpose(1, 2))
    dk = torch.matmul(d.transpose(2, 3), _grouped(q, Hk))
    return _ungrouped(dq, T), dk.transpose(1, 2), dv.transpose(1, 2)


def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind == "ranges":
        return _ranges(s["mask"], s["done"], s["tokens"], s["mode"], s["prefix"], (s["rows"], s["cols"]) if s["rows"] else None)
    dtype = DTYPES[s["dtype"]]
    if kind == "norm":
        c, si = _rotation(s)
        q, k = _norm_rotate(s["q"], s["wq"], c, si).to(dtype), _norm_rotate(s["k"], s["wk"], c, si).to(dtype)
        if s["append"]:
            at = s["slots"].long()
            row = torch.arange(s["B"], device=at.device)[:, None]
            s["k_cache"][row, at] = k
            s["v_cache"][row, at] = s["v"]
            return q, s["k_cache"], s["v_cache"]
        dq, dwq = _norm_rotate_grad(s["gq"], s["q"], s["wq"], c, si)
        dk, dwk = _norm_rotate_grad(s["gk"], s["k"], s["wk"], c, si)
        return q, k, dq.to(dtype), dk.to(dtype), dwq, dwk
    if kind == "step":
        return _ungrouped(_attend(s, s["hi"] - 1)[0], s["T"]).to(dtype)
    place = (torch.arange(s["T"], device="cuda") + s["S"] - s["T"])[None]
    out, lse, p, slope = _attend(s, place)
    if not s["train"]:
        return _ungrouped(out, s["T"]).to(dtype), lse
    dq, dk, dv = _attend_grad(s, out, p, slope)
    return _ungrouped(out, s["T"]).to(dtype), lse, dq.to(dtype), dk.to(dtype), dv.to(dtype)


# ---- the framework's operators -----------------------------------------------------------------------------

def _run_own(s):
    from gear_amd import ops
    kind = s["kind"]
    if kind == "ranges":
        return ops.token_ranges(s["mask"], s["done"], tokens_per_step=s["tokens"], mode=s["mode"], prefix=s["prefix"],
                                grid=(s["rows"], s["cols"]) if s["rows"] else None)
    if kind == "norm":
        how = (s["pos"], s["freqs"], _sections(s), s["wq"], s["wk"])
        if s["append"]:
            q = ops.norm_rotate_append(s["q"], s["k"], s["v"], *how, slots=s["slots"], k_cache=s["k_cache"],
                                       v_cache=s["v_cache"], eps=EPS)
            return q, s["k_cache"], s["v_cache"]
        q, k = ops.norm_rotate(s["q"], s["k"], *how, eps=EPS)
        return (q, k) + tuple(ops.norm_rotate_backward(s["gq"], s["gk"], s["q"], s["k"], *how, eps=EPS))
    form = dict(cap=s["cap"], slopes=s["slopes"])
    if kind == "step":
        return ops.range_attention_step(s["q"], s["k"], s["v"], s["lo"], s["hi"], **form)
    out, lse = ops.range_attention(s["q"], s["k"], s["v"], s["lo"], s["hi"], **form)
    if not s["train"]:
        return out, lse
    return (out, lse) + tuple(ops.range_attention_backward(s["gout"], s["q"], s["k"], s["v"], out, lse, s["lo"], s["hi"],
                                                           **form))


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    kind, B = case["kind"], case["B"]
    if kind == "ranges":
        tokens = B * case["S"] * case["tokens"]
        return {"bytes": 2 * B * case["S"] + tokens * (20 if case["rows"] else 12), "flops": 0}
    Hq, Hk, D, T = case["Hq"], case["Hk"], case["D"], case["T"]
    size = 4 if case["dtype"] == "float32" else 2
    if kind == "norm":
        rows = B * T * (Hq + Hk) * D
        pos = B * T * len(_sections(case)) * 4
        if case["append"]:
            return {"bytes": size * (2 * rows + 2 * B * T * Hk * D) + pos, "flops": 10 * rows}
        return {"bytes": size * 5 * rows + 2 * pos, "flops": 30 * rows}
    if kind == "step":  # caches are filled to a length between T and L, a third of them begin later
        keys = B * (T + (case["L"] - T) / 2) * 0.955
        return {"bytes": size * (2 * keys * Hk * D + 2 * B * T * Hq * D), "flops": 4 * D * keys * T * Hq}
    S = case["S"]
    mask, done = _steps(case, 0, "cpu")
    lo, hi, _ = _ranges(mask, done, case["tokens"], case["mode"], case["prefix"], None)
    pairs = int((hi[:, S - T:] - lo[:, S - T:]).long().sum()) * Hq
    qs, ks = B * T * Hq * D * size, B * S * Hk * D * size
    if not case["train"]:
        return {"bytes": 2 * qs + 2 * ks + 4 * B * T * (2 + Hq), "flops": 4 * D * pairs}
    # forward and backward; the backward needs queries, keys, values and its own output again
    return {"bytes": 6 * qs + 6 * ks + 8 * B * T * (2 + Hq), "flops": 14 * D * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def _exact_norm(s):
    """By complex numbers: a pair is a + ib, the rotation a product with exp(i angle); gradients by autograd."""
    half, sections = s["D"] // 2, _sections(s)
    angle = torch.zeros(s["B"], s["T"], half, dtype=torch.float64, device="cuda")
    start = 0
    for axis, n in enumerate(sections):
        angle[..., start:start + n] = s["pos"][..., axis, None].double() * s["freqs"][start:start + n]
        start += n
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]

    def f(x, w):
        y = w * x / torch.sqrt((x * x).sum(-1, keepdim=True) / s["D"] + EPS)
        z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    outs, grads, weights = [], [], []
    for name in ("q", "k"):
        x, w = s[name].double(), s["w" + name].double()
        if s["train"]:
            x, w = x.requires_grad_(), w.requires_grad_()
            y = f(x, w)
            gx, gw = torch.autograd.grad(y, (x, w), s["g" + name].double())
            grads.append(gx)
            weights.append(gw)
        else:
            y = f(x, w)
        outs.append(y.detach())
    if not s["append"]:
        return tuple(outs + grads + weights)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    at = s["slots"].tolist()
    for b in range(s["B"]):
        for t in range(s["T"]):
            k_cache[b, at[b][t]] = outs[1][b, t]
            v_cache[b, at[b][t]] = s["v"][b, t].double()
    return outs[0], k_cache, v_cache


def _exact_attention(s, train, place):
    B, T, Hq, D = s["q"].shape
    S, Hk = s["k"].shape[1:3]
    G = Hq // Hk
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, Hq, T, dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk, dv = (torch.zeros(B, S, Hk, D, dtype=torch.float64, device="cuda") for _ in range(2))
    group = max(1, min(B, int(2e7) // (T * S)))
    at = torch.arange(S, device="cuda")
    for b in range(0, B, group):
        e = min(B, b + group)
        hidden = (at[None, None] < s["lo"][b:e, :, None]) | (at[None, None] >= s["hi"][b:e, :, None])
        empty = hidden.all(-1, keepdim=True)
        for h in range(Hq):
            q, k, v = (x.double().requires_grad_() for x in (s["q"][b:e, :, h], s["k"][b:e, :, h // G], s["v"][b:e, :, h // G]))
            x = q @ k.transpose(1, 2) / math.sqrt(D)
            if s["cap"]:
                x = s["cap"] * torch.tanh(x / s["cap"])
            if s["slopes"] is not None:
                x = x - float(s["slopes"][h]) * (place[b:e, :, None] - at).abs()
            x = torch.where(hidden, torch.full_like(x, -1e300), x)
            z = torch.logsumexp(x, -1, keepdim=True)
            y = torch.where(empty, torch.zeros_like(z), torch.exp(x - z)) @ v
            out[b:e, :, h], lse[b:e, h] = y.detach(), torch.where(empty, float("-inf"), z.detach())[..., 0]
            if train:
                a, c, d = torch.autograd.grad(y, (q, k, v), s["gout"][b:e, :, h].double())
                dq[b:e, :, h] = a
                dk[b:e, :, h // G] += c
                dv[b:e, :, h // G] += d
    return (out, lse, dq, dk, dv) if train else (out, lse)


def exact(case, seed):
    kind = case["kind"]
    if kind == "ranges":
        return None
    s = prepare(case, seed)
    if kind == "norm":
        return _exact_norm(s)
    place = s["hi"].long() - 1 if kind == "step" else \
        (torch.arange(case["T"], device="cuda") + case["S"] - case["T"]).expand(case["B"], case["T"])
    if kind == "step":
        return _exact_attention(s, False, place)[0]
    return _exact_attention(s, case["train"], place)
