"""The operators between a batch of windows and a sequence model, plainly and in 64 bits, with bounds of the error that
16-bit inputs and outputs allow.  Independent of gear_amd."""
import math

import numpy as np
import torch

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}  # of one rounding
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half the smallest step
FLUSHED = 2.0 ** -126  # 32-bit exponentials (and bfloat16 operands) below the smallest normal number become 0


def token_ranges(mask, done, tokens, mode, prefix, grid):
    """numpy, one step after the other."""
    B, S = mask.shape
    T = S * tokens
    lo, hi = np.zeros((B, T), np.int32), np.zeros((B, T), np.int32)
    pos = np.zeros((B, T, 3 if grid else 1), np.int32)
    for b in range(B):
        s = 0
        while s < S:
            if not mask[b, s]:
                s += 1
                continue
            e = s
            while not done[b, e] and e + 1 < S and mask[b, e + 1]:
                e += 1
            e += 1
            for x in range(s, e):
                for u in range(tokens):
                    i = x * tokens + u
                    lo[b, i] = s * tokens
                    hi[b, i] = {"causal": i + 1, "step": (x + 1) * tokens, "document": e * tokens}[mode]
                    if prefix:
                        hi[b, i] = max(hi[b, i], min(s + prefix, e) * tokens)
                    pos[b, i] = (x - s, u // grid[1], u % grid[1]) if grid else (x - s,)
            s = e
    return lo, hi, pos


def norm_rotate(x, w, pos, freqs, sections, eps):
    """float64 in, float64 out; differentiable."""
    D = x.shape[-1]
    angle = torch.zeros(x.shape[:2] + (D // 2,), dtype=torch.float64, device=x.device)
    at = 0
    for axis, n in enumerate(sections):
        angle[..., at:at + n] = pos[..., axis, None].double() * freqs[at:at + n]
        at += n
    c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


class Attention:
    """out, lse and, with dout, dq, dk, dv in 64 bits, and for each a bound of the error of an implementation that rounds
    the probabilities (and their gradients) once to the inputs' type, works from the rounded out, and rounds its result."""

    def __init__(self, q, k, v, lo, hi, scale=None, cap=0.0, slopes=None, dout=None, place=None):
        dtype = q.dtype
        u, tiny = UNIT[dtype], TINY[dtype]
        B, T, H, D = q.shape
        S, HK = k.shape[1:3]
        scale = D ** -0.5 if scale is None else scale
        # what no range reaches is not part of the definition: nothing of it may be read
        at = torch.arange(S, device=q.device)
        l, h = lo.clamp(min=0)[..., None], hi.clamp(max=S)[..., None]
        seen = ((at >= l) & (at < h))[:, None]  # [B, 1, T, S]
        some = seen.any(-1)[:, 0, :, None, None]
        used = seen.any(2)[:, 0, :, None, None]
        heads = lambda x: x.double().permute(0, 2, 1, 3).contiguous()  # noqa: E731
        q = heads(torch.where(some, q, torch.zeros_like(q)))
        k, v = (heads(torch.where(used, x, torch.zeros_like(x))).repeat_interleave(H // HK, 1) for x in (k, v))
        x = q @ k.transpose(2, 3) * scale
        size = (q.abs() @ k.abs().transpose(2, 3) * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
        slope = 1.0
        if cap:
            t = torch.tanh(x / cap)
            x, slope = cap * t, 1 - t * t
        if slopes is not None:
            p = (torch.arange(T, device=q.device) + S - T).expand(B, T) if place is None else place.long()
            bias = slopes.double()[None, :, None, None] * (p[:, None, :, None] - at).abs()
            x = x - bias
            size = size + bias.masked_fill(~seen, 0).amax(-1, keepdim=True)
        x = x.masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True).clamp(min=-1e300)
        e = torch.exp(x - top)
        total = e.sum(-1, keepdim=True)
        p = torch.where(total > 0, e / total, 0.0)
        # 32-bit scores: a relative error of p, sums of D products, the exponent and the table of exp2
        fine = 2.0 ** -24 * (8 + math.sqrt(D)) * (size + cap + 16)
        back = lambda y: y.permute(0, 2, 1, 3)  # noqa: E731
        out = p @ v
        self.out, self.lse = back(out), (torch.log(total) + top).squeeze(-1)
        self.lse = torch.where(total.squeeze(-1) > 0, self.lse, -math.inf)
        weight = p @ v.abs()
        self.out_bound = back((u + fine) * weight * 1.01 + u * out.abs() + tiny * (1 + seen.double() @ v.abs()))
        self.lse_bound = (fine.squeeze(-1) + 2.0 ** -23 * self.lse.abs().clamp(max=1e30)) + 2e-7
        if dout is None:
            return
        g = heads(torch.where(some, dout, torch.zeros_like(dout)))
        dp = g @ v.transpose(2, 3)
        delta = (g * out).sum(-1, keepdim=True)
        ds = p * (dp - delta) * slope
        # of delta: out was rounded to the type (and has its own error); of dp: a 32-bit sum
        off = ((g.abs() * (self.out_bound.permute(0, 2, 1, 3))).sum(-1, keepdim=True) +
               2.0 ** -24 * 2 * math.sqrt(D) * (g.abs() @ v.abs().transpose(2, 3)).amax(-1, keepdim=True))
        wrong = (u + 2 * fine) * ds.abs() + p * off + (tiny + FLUSHED * (1 + (dp - delta).abs())) * seen
        fold = lambda y: back(y.view(B, HK, H // HK, S, D).sum(2))  # noqa: E731
        dq, dk, dv = ds @ k * scale, ds.transpose(2, 3) @ q * scale, p.transpose(2, 3) @ g
        self.dq, self.dk, self.dv = back(dq), fold(dk), fold(dv)
        self.dq_bound = back(1.01 * scale * (wrong @ k.abs())) + u * self.dq.abs() + tiny
        self.dk_bound = fold(1.01 * scale * (wrong.transpose(2, 3) @ q.abs())) + u * self.dk.abs() + tiny
        pw = (u + fine) * p + (tiny * 2.0 ** -8 + FLUSHED) * seen
        self.dv_bound = fold(1.01 * (pw.transpose(2, 3) @ g.abs())) + u * self.dv.abs() + tiny


def worst(got, ref, bound):
    """The largest error as a share of its bound; infinite where a value is not finite and the reference is."""
    same = (got.double() == ref) | (torch.isnan(got) & torch.isnan(ref))
    share = (got.double() - ref).abs() / bound
    share = torch.where(same, torch.zeros_like(share), torch.where(torch.isfinite(share), share, math.inf))
    return float(share.max()) if share.numel() else 0.0
