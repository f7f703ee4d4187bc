"""Sequence models over the loader's windows: the operators of gear_amd.ops as differentiable functions, and a
small causal model of observations and actions that uses them as they are meant to be used together.

    masks, done column --token_ranges--> ranges of keys, positions
    queries, keys      --norm_rotate--->  range_attention          (a batch of windows, with gradients)
                       --norm_rotate_append--> range_attention_step  (the next step of rollouts, from caches)

No counterpart in the reference, whose loader hands its batches to models outside of it
(gear/loader/offline_loader.py:155-204)."""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import ops


def _rows(t):
    """A gradient as it comes (expanded, transposed), in rows that the operators take."""
    size = t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * size % 16 == 0 for s in t.stride()[:-1]):
        return t
    return t.contiguous()


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, pos, freqs, sections, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, pos, freqs)
        ctx.form = (sections, eps)
        return ops.norm_rotate(q, k, pos, freqs, sections, q_weight, k_weight, eps=eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, pos, freqs = ctx.saved_tensors
        sections, eps = ctx.form
        return ops.norm_rotate_backward(_rows(dq_out), _rows(dk_out), q, k, pos, freqs, sections, q_weight, k_weight,
                                        eps=eps) + (None,) * 4


def norm_rotate(q, k, pos, freqs, sections, q_weight=None, k_weight=None, *, eps=1e-6):
    """gear_amd.ops.norm_rotate with gradients of q, k and the weights."""
    return _NormRotate.apply(q, k, q_weight, k_weight, pos, freqs, tuple(sections), eps)


class _RangeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lo, hi, scale, cap, slopes):
        out, lse = ops.range_attention(q, k, v, lo, hi, scale=scale, cap=cap, slopes=slopes)
        ctx.save_for_backward(q, k, v, out, lse, lo, hi, slopes)
        ctx.form = (scale, cap)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, lo, hi, slopes = ctx.saved_tensors
        scale, cap = ctx.form
        return ops.range_attention_backward(_rows(dout), q, k, v, out, lse, lo, hi, scale=scale, cap=cap,
                                            slopes=slopes) + (None,) * 5


def range_attention(q, k, v, lo, hi, *, scale=None, cap=0.0, slopes=None):
    """The out of gear_amd.ops.range_attention with gradients of q, k and v (slopes are constants)."""
    if slopes is not None and slopes.requires_grad:
        raise ValueError("slopes have no gradient: pass them detached")
    return _RangeAttention.apply(q, k, v, lo, hi, scale, cap, slopes)


class _Block(nn.Module):
    def __init__(self, width, heads, kv_heads):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.before, self.between = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * self.dim, bias=False)
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(self.dim)), nn.Parameter(torch.ones(self.dim))
        self.out = nn.Linear(width, width, bias=False)
        self.mlp = nn.Sequential(nn.Linear(width, 4 * width), nn.GELU(), nn.Linear(4 * width, width))

    def split(self, x, dtype):
        qkv = self.qkv(self.before(x)).to(dtype).view(*x.shape[:2], -1, self.dim)
        return qkv.split([self.heads, self.kv_heads, self.kv_heads], 2)

    def weights(self, dtype):
        """Of the norm, in a type that it takes beside rows of `dtype`: theirs, or 32 bits."""
        return [w if w.dtype in (dtype, torch.float32) else w.float() for w in (self.q_weight, self.k_weight)]

    def rest(self, x, attended):
        x = x + self.out(attended.flatten(2).to(x.dtype))
        return x + self.mlp(self.between(x))


class Rollouts:
    """The caches of a batch of rollouts: per layer keys and values of up to `tokens` tokens, and how many are there.
    A step is two tokens, the first of a rollout one."""

    def __init__(self, model, batch, tokens):
        self.tokens, self.taken = tokens, 0  # (known here as well: no step waits for the GPU to compare them)
        at = dict(dtype=model.dtype, device=model.freqs.device)
        shape = (len(model.blocks), 2, batch, tokens, model.blocks[0].kv_heads, model.blocks[0].dim)
        self.caches = torch.zeros(shape, **at)
        self.length = torch.zeros(batch, 1, dtype=torch.int32, device=at["device"])
        self.time = torch.zeros(batch, 1, dtype=torch.int32, device=at["device"])

    def restart(self):
        """All rollouts begin anew, in the same caches."""
        self.taken = 0
        self.length.zero_()
        self.time.zero_()


class WindowModel(nn.Module):
    """Predicts each step's action from the window's observations and actions up to it.

    A step is two tokens, observation then action; a token sees its document (the window's valid steps up to the
    last end of an episode) up to itself.  Positions have the axes (time, row, column) of a grid of 1 x 2 tokens a step.
    The projections run in the parameters' type (any, and what comes in has it), attention in `dtype`."""

    TOKENS = 2

    def __init__(self, observation, action, width=128, heads=4, kv_heads=2, layers=2, cap=30.0, dtype=torch.bfloat16):
        super().__init__()
        self.dtype, self.cap = dtype, cap
        self.embed = nn.ModuleList([nn.Linear(observation, width), nn.Linear(action, width)])
        self.blocks = nn.ModuleList(_Block(width, heads, kv_heads) for _ in range(layers))
        self.head = nn.Sequential(nn.LayerNorm(width), nn.Linear(width, action))
        pairs = width // heads // 2
        self.sections = (pairs - pairs // 4, 0, pairs // 4)
        self.register_buffer("freqs", ops.rotation_freqs(self.sections, device="cpu"), persistent=False)

    def _apply(self, *args, **kwargs):
        """Casts are for the parameters: the frequencies stay in 64 bits, and go along to another device."""
        freqs = self.freqs
        super()._apply(*args, **kwargs)
        device = self.freqs.device
        self.freqs = ops.rotation_freqs(self.sections, device=device) if freqs.is_meta else freqs.to(device)
        return self

    def forward(self, observations, actions, mask, done):
        """observations [batch, steps, ...], actions, the loader's mask, the done column -> actions [batch, steps, ...]."""
        batch, steps = mask.shape
        lo, hi, pos = ops.token_ranges(mask, done, tokens_per_step=self.TOKENS, mode="causal", grid=(1, self.TOKENS))
        x = torch.stack([self.embed[0](observations.flatten(2)), self.embed[1](actions.flatten(2))], 2).flatten(1, 2)
        for block in self.blocks:
            q, k, v = block.split(x, self.dtype)
            q, k = norm_rotate(q, k, pos, self.freqs, self.sections, *block.weights(self.dtype))
            x = block.rest(x, range_attention(q, k, v, lo, hi, cap=self.cap))
        return self.head(x.view(batch, steps, self.TOKENS, -1)[:, :, 0])

    @torch.no_grad()
    def step(self, rollouts, observation, last_action=None):
        """The next action of every rollout, from its newest observation [batch, ...] and the action before it (None: the
        first step)."""
        new = 1 if last_action is None else 2
        if rollouts.taken + new > rollouts.tokens:
            raise ValueError("the rollouts' caches of %d tokens hold %d: no room for %d more"
                             % (rollouts.tokens, rollouts.taken, new))
        x = [self.embed[0](observation)]
        column = [torch.zeros_like(rollouts.time)]
        time = [rollouts.time]
        if last_action is not None:  # its token comes first: it belongs to the step before
            x, column, time = [self.embed[1](last_action)] + x, [column[0] + 1] + column, [rollouts.time - 1] + time
        x = torch.stack(x, 1)
        pos = torch.stack([torch.cat(time, 1), torch.zeros_like(torch.cat(time, 1)), torch.cat(column, 1)], 2)
        slots = rollouts.length + torch.arange(x.shape[1], dtype=torch.int32, device=x.device)
        lo, hi = torch.zeros_like(slots), slots + 1
        for block, (keys, values) in zip(self.blocks, rollouts.caches):
            q, k, v = block.split(x, self.dtype)
            q = ops.norm_rotate_append(q, k, v, pos, self.freqs, self.sections, *block.weights(self.dtype), slots=slots,
                                       k_cache=keys, v_cache=values)
            x = block.rest(x, ops.range_attention_step(q, keys, values, lo, hi, cap=self.cap))
        rollouts.taken += new
        rollouts.length += new
        rollouts.time += 1
        return self.head(x[:, -1])
