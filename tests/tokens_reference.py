"""The operators of token models, plainly and in 64 bits, with bounds of the error of an implementation that works in 32 bits
and rounds its results once.  Independent of gear_amd."""
import math

import torch

from sequence_reference import TINY, UNIT

E = 2.0 ** -24  # one rounding in 32 bits
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rounded(ref, dtype):
    """One rounding of a result; 32-bit subnormals may be flushed."""
    return UNIT[dtype] * ref.abs() + TINY[dtype] + 2.0 ** -126


def embed(tokens, table, scale):
    inside = (tokens >= 0) & (tokens < table.shape[0])
    ref = torch.where(inside[..., None], table.double()[tokens.clamp(0, max(table.shape[0] - 1, 0)).long()] * scale, 0.0)
    # the product is rounded to 32 bits, then to the type
    return ref, rounded(ref, table.dtype) + E * ref.abs()


def embed_backward(dout, tokens, vocab, scale):
    """n rows of a token are added in 32 bits in some order: n - 1 roundings of at most the sum of sizes, and the product."""
    t, d = tokens.reshape(-1).long(), dout.double().reshape(-1, dout.shape[-1])
    inside = (t >= 0) & (t < vocab)
    t, d = t[inside], d[inside]
    ref, size = (torch.zeros(vocab, d.shape[1], dtype=torch.float64, device=d.device).index_put_((t,), x * scale, accumulate=True)
                 for x in (d, d.abs()))
    size = size.abs()
    count = torch.bincount(t, minlength=vocab).double()[:, None]
    return ref, rounded(ref, dout.dtype) + E * (count + 1) * size * (1 + 2.0 ** -10)


class LayerNorm:
    """Of u as it is stored.  32-bit sums over a row: at most 16 elements of a lane and 10 levels of lanes, 26 roundings of
    the mean size; deviations, products and the root (1 unit) a few more: 64 units cover them."""

    def __init__(self, u, w, b, eps, dy=None, dsum=None):
        dtype, W = u.dtype, u.shape[-1]
        u = u.double().reshape(-1, W)
        one, zero = torch.ones(W, dtype=torch.float64, device=u.device), torch.zeros(W, dtype=torch.float64, device=u.device)
        w, b = (one if w is None else w.double()), (zero if b is None else b.double())
        c = u - u.mean(-1, keepdim=True)
        r = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
        n = c * r
        off = r * u.abs().mean(-1, keepdim=True)  # what an error of the mean is to n
        self.y = n * w + b
        self.y_bound = rounded(self.y, dtype) + 64 * E * (w.abs() * (n.abs() + off) + b.abs())
        if dy is None:
            return
        dy = dy.double().reshape(-1, W)
        mean = lambda x: x.mean(-1, keepdim=True)  # noqa: E731
        h = dy * w
        self.dx = r * (h - mean(h) - n * mean(h * n))
        size = r * (h.abs() + mean(h.abs()) + (n.abs() + off) * mean(h.abs() * (n.abs() + off)))
        if dsum is not None:
            self.dx = self.dx + dsum.double().reshape(-1, W)
            size = size + dsum.double().reshape(-1, W).abs()
        self.dx_bound = rounded(self.dx, dtype) + 64 * E * size
        rows = u.shape[0]
        self.dw, self.db = (dy * n).sum(0), dy.sum(0)
        self.dw_error = E * (rows + 64) * (dy.abs() * (n.abs() + off)).sum(0)
        self.db_error = E * (rows + 64) * dy.abs().sum(0)


class LogProbs:
    """x -> statistics of softmax(scale * x), -inf not allowed, nor rows of the lowest numbers.  d = scale (x - max) has three roundings; S and A are sums
    of at most 160 elements of a lane and 20 levels of lanes and parts."""

    def __init__(self, x, scale):
        x, self.scale = x.double(), scale
        self.z = torch.where(x.amax(-1, keepdim=True) < -1e30, -math.inf, x) * scale
        top = self.z.amax(-1, keepdim=True)
        self.none = (top == -math.inf)[:, 0]
        shift = torch.where(top == -math.inf, 0.0, top)
        d = self.z - shift
        e = torch.exp(d)
        s = e.sum(-1, keepdim=True)
        self.d = torch.where(e > 0, d, 0.0)
        self.p = torch.where(s > 0, e / s, 0.0)
        self.lse = (torch.log(s) + shift)[:, 0]
        self.logp = self.z - self.lse[:, None]
        self.finite_logp = torch.where(self.p > 0, self.logp, 0.0)
        self.entropy = -(self.p * self.finite_logp).sum(-1)
        size = (self.p * self.d.abs()).sum(-1)
        square = (self.p * self.d.square()).sum(-1)
        self.s_error = E * (200 + 4 * size + 4 * torch.log(s)[:, 0].abs().clamp(max=100))
        self.lse_bound = self.s_error + 3 * E * torch.where(self.none, 0.0, self.lse).abs()
        self.entropy_bound = 2 * self.s_error + E * (200 * size + 8 * square + 4)

    def logp_bound(self, logp, d):
        return self.s_error + E * (4 * d.abs() + 2 * logp.abs() + 4)

    def gradient(self, alpha, beta, add, dtype, lse, extra):
        """scale (p (alpha + beta log p) + add), p from the lse that it is given in 32 bits; alpha and beta are off by up
        to 16 units of extra."""
        value = self.p * (alpha + beta * self.finite_logp) + add
        seen = self.p > 0
        z = torch.where(seen, self.z, 0.0)
        off = E * (4 * (z.abs() + torch.where(self.none, 0.0, lse).abs()[:, None]) + 12) + self.lse_bound[:, None]
        size = self.p * ((1 + off) * off * (alpha.abs() + beta.abs() * (1 + self.finite_logp.abs())) + E * 16 * extra)
        ref = self.scale * value
        return ref, rounded(ref, dtype) + self.scale * (size + E * 4 * add.abs() + 2.0 ** -120 * (1 + extra))


def order(x, k):
    """The k largest of rows, the lower index first among equals, NaN before all."""
    return torch.sort(x.double() + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]


def teacher(top_tokens, top_logits, vocab):
    there = (top_tokens >= 0) & (top_tokens < vocab)
    t = torch.where(there, top_logits.double(), -math.inf)
    top = t.amax(-1, keepdim=True)
    some = (top > -math.inf)[:, 0]
    e = torch.exp(t - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    q = torch.where(total > 0, e / total, 0.0)
    # 64 entries are added
    error = q * E * (80 + 4 * torch.where(q > 0, (t - top).abs(), 0.0))
    return q, error, some
