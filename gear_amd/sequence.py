"""Sequence models over the loader's windows: the operators of gear_amd.ops as differentiable functions, and a
small causal model of observations and actions that uses them as they are meant to be used together.

    masks, done column --token_ranges--> ranges of keys, positions
    queries, keys      --norm_rotate--->  range_attention          (a batch of windows, with gradients)
                       --norm_rotate_append--> range_attention_step  (the next step of rollouts, from caches)

and the same for windows whose observations and actions are tokens:

    tokens --embed_tokens--> [layer_norm, attention, layer_norm with the sum]... --> logits
    logits --token_log_probs--> log probabilities of actions, entropies, the best few (acting; a teacher's say)
           --distill----------> the divergence from a teacher's best few

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


def _matrix(t):
    """A gradient as it comes, with rows at one stride."""
    lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    fits = t.stride(-1) == 1 and all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:]))
    return t if fits else t.contiguous()


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.save_for_backward(tokens)
        ctx.form = (table.shape[0], scale)
        return ops.embed_tokens(tokens, table, scale=scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        vocab, scale = ctx.form
        return None, ops.embed_tokens_backward(_matrix(dout), ctx.saved_tensors[0], vocab, scale=scale), None


def embed_tokens(tokens, table, *, scale=1.0):
    """gear_amd.ops.embed_tokens with the gradient of the table."""
    return _EmbedTokens.apply(tokens, table, scale)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight, bias)
        ctx.eps = eps
        return ops.layer_norm(x, weight, bias, eps=eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        return ops.layer_norm_backward(_matrix(dy), x, weight, bias, eps=ctx.eps) + (None,)


class _SumNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, total = ops.layer_norm(x, weight, bias, residual=residual, eps=eps)
        ctx.save_for_backward(total, weight, bias)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum):
        total, weight, bias = ctx.saved_tensors
        if dy is None:
            return dsum, dsum, None, None, None
        dx, dweight, dbias = ops.layer_norm_backward(_matrix(dy), total, weight, bias,
                                                     dsum=None if dsum is None else _matrix(dsum), eps=ctx.eps)
        return dx, dx, dweight, dbias, None


def layer_norm(x, weight=None, bias=None, *, residual=None, eps=1e-5):
    """gear_amd.ops.layer_norm with gradients of x, the residual, the weight and the bias."""
    if residual is None:
        return _LayerNorm.apply(x, weight, bias, eps)
    return _SumNorm.apply(x, residual, weight, bias, eps)


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, scale, top):
        outs = ops.token_log_probs(logits, tokens, scale=scale, top=top)
        ctx.save_for_backward(logits, tokens, outs[2], outs[1])
        ctx.scale = scale
        ctx.mark_non_differentiable(*(t for t in outs[2:] if t is not None))
        ctx.set_materialize_grads(False)
        return outs

    @staticmethod
    @once_differentiable
    def backward(ctx, dlog_probs, dentropy, *_):
        if dlog_probs is None and dentropy is None:
            return None, None, None, None
        logits, tokens, lse, entropy = ctx.saved_tensors
        dlog_probs, dentropy = (None if t is None else t.contiguous() for t in (dlog_probs, dentropy))
        return ops.token_log_probs_backward(dlog_probs, dentropy, logits, tokens, lse, entropy, scale=ctx.scale), None, None, None


def token_log_probs(logits, tokens=None, *, scale=1.0, top=0):
    """gear_amd.ops.token_log_probs with the gradient of the logits through the log probabilities and the entropy (lse
    and the best tokens are constants)."""
    return _TokenLogProbs.apply(logits, tokens, scale, top)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_tokens, top_logits, scale):
        loss, lse = ops.distill(logits, top_tokens, top_logits, scale=scale)
        ctx.save_for_backward(logits, top_tokens, top_logits, lse)
        ctx.scale = scale
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        return ops.distill_backward(dloss.contiguous(), *ctx.saved_tensors, scale=ctx.scale), None, None, None


def distill(logits, top_tokens, top_logits, *, scale=1.0):
    """The loss of gear_amd.ops.distill with the gradient of the logits (the teacher is a constant)."""
    if top_logits.requires_grad:
        raise ValueError("top_logits have no gradient: pass them detached")
    return _Distill.apply(logits, top_tokens, top_logits, scale)


class _Norm(nn.LayerNorm):
    """nn.LayerNorm by layer_norm; with a residual: (y, the sum)."""

    def forward(self, x, residual=None):
        return layer_norm(x, self.weight, self.bias, residual=residual, eps=self.eps)


class _Block(nn.Module):
    def __init__(self, width, heads, kv_heads, norm=nn.LayerNorm):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.before, self.between = norm(width), norm(width)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * self.dim, bias=False)
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(self.dim)), nn.Parameter(torch.ones(self.dim))
        self.out = nn.Linear(width, width, bias=False)
        self.mlp = nn.Sequential(nn.Linear(width, 4 * width), nn.GELU(), nn.Linear(4 * width, width))

    def split(self, x, dtype):
        return self.project(self.before(x), dtype)

    def project(self, y, dtype):
        qkv = self.qkv(y).to(dtype).view(*y.shape[:2], -1, self.dim)
        return qkv.split([self.heads, self.kv_heads, self.kv_heads], 2)

    def weights(self, dtype):
        """Of the norm, in a type that it takes beside rows of `dtype`: theirs, or 32 bits."""
        return [w if w.dtype in (dtype, torch.float32) else w.float() for w in (self.q_weight, self.k_weight)]

    def rest(self, x, attended):
        x = x + self.out(attended.flatten(2).to(x.dtype))
        return x + self.mlp(self.between(x))


class Rollouts:
    """The caches of a batch of rollouts: per layer keys and values of up to `tokens` tokens, and how many are there.
    A step is as many tokens as the model has a step, the first of a rollout one less."""

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


class _Positions(nn.Module):
    """A model whose heads are rotated by their tokens' positions."""

    def positions(self, dim):
        pairs = dim // 2
        self.sections = (pairs - pairs // 4, 0, pairs // 4)
        self.register_buffer("freqs", ops.rotation_freqs(self.sections, device="cpu"), persistent=False)

    def _apply(self, *args, **kwargs):
        """Casts are for the parameters: the frequencies stay in 64 bits, and go along to another device."""
        freqs = self.freqs
        super()._apply(*args, **kwargs)
        device = self.freqs.device
        self.freqs = ops.rotation_freqs(self.sections, device=device) if freqs.is_meta else freqs.to(device)
        return self


class WindowModel(_Positions):
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
        self.positions(width // heads)

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


class TokenModel(_Positions):
    """A causal policy over tokens: a step is `step` of them, its observation's (in bins, patches, words) and its action
    last; from the tokens up to an action comes the distribution of that action.  Ends of episodes and padding are
    those of WindowModel.  Everything runs in the parameters' type (32, 16 bits or bfloat16), attention in `dtype`; under
    autocast the projections and the logits in its type."""

    def __init__(self, vocab, step, width=128, heads=4, kv_heads=2, layers=2, cap=30.0, dtype=torch.bfloat16):
        super().__init__()
        if step < 2:
            raise ValueError("a step needs two tokens at least, an observation's and its action")
        self.step_tokens, self.width, self.dtype, self.cap = step, width, dtype, cap
        self.table = nn.Parameter(torch.randn(vocab, width) * width ** -0.5)
        self.blocks = nn.ModuleList(_Block(width, heads, kv_heads, _Norm) for _ in range(layers))
        self.norm = _Norm(width)
        self.head = nn.Linear(width, vocab, bias=False)
        self.positions(width // heads)

    @staticmethod
    def _norm(norm, x, residual=None):
        if isinstance(norm, _Norm) or residual is None:
            return norm(x) if residual is None else norm(x, residual)
        total = x + residual  # another module in a norm's place
        return norm(total), total

    def _logits(self, tokens, attend, actions):
        """tokens [batch, tokens]; attend(layer, block, q, k, v) -> [batch, tokens, heads, dim]; actions(x) picks the rows
        that an action is read from."""
        x = embed_tokens(tokens, self.table, scale=self.width ** 0.5)
        y = self._norm(self.blocks[0].before, x)
        for i, block in enumerate(self.blocks):
            attended = attend(i, block, *block.project(y, self.dtype)).flatten(2).to(x.dtype)
            # (autocast's results in 16 bits are added to in the table's type, as its sums are)
            y, x = self._norm(block.between, block.out(attended).to(x.dtype), x)
            more = block.mlp(y).to(x.dtype)
            if i + 1 < len(self.blocks):
                y, x = self._norm(self.blocks[i + 1].before, more, x)
        return self.head(self._norm(self.norm, actions(more), actions(x))[0])

    def forward(self, tokens, mask, done):
        """tokens [batch, steps, step], the loader's mask, the done column -> logits [batch, steps, vocab] of every
        step's action."""
        batch, steps, n = tokens.shape
        lo, hi, pos = ops.token_ranges(mask, done, tokens_per_step=n, mode="causal", grid=(1, n))

        def attend(_, block, q, k, v):
            q, k = norm_rotate(q, k, pos, self.freqs, self.sections, *block.weights(self.dtype))
            return range_attention(q, k, v, lo, hi, cap=self.cap)

        return self._logits(tokens.flatten(1).contiguous(), attend, lambda x: x.view(batch, steps, n, -1)[:, :, n - 2])

    @staticmethod
    def taken(tokens, mask):
        """The actions of windows, none (-1) in their padding."""
        return tokens[:, :, -1].masked_fill(mask == 0, -1)

    def log_probs(self, tokens, mask, done, *, scale=1.0, top=0):
        """token_log_probs of the windows' actions."""
        return token_log_probs(self(tokens, mask, done), self.taken(tokens, mask), scale=scale, top=top)

    def distilled(self, teacher, tokens, mask, done, *, count=8, scale=1.0):
        """distill [batch, steps] from the best `count` actions of a teacher (a TokenModel too) on the same windows."""
        with torch.no_grad():
            best = teacher.log_probs(tokens, mask, done, scale=scale, top=count)
        return distill(self(tokens, mask, done), best[4], best[3], scale=scale)

    @torch.no_grad()
    def step(self, rollouts, observation, last_action=None, *, top=1, scale=1.0):
        """The next action of every rollout, from the tokens of its newest observation [batch, step - 1] and the action
        before it [batch] (None: the first step): (entropy [batch], top_log_probs, top_tokens [batch, top])."""
        n = self.step_tokens
        tokens, column, time = observation, torch.arange(n - 1, device=observation.device), rollouts.time.expand(-1, n - 1)
        if last_action is not None:  # its token comes first: it belongs to the step before
            tokens = torch.cat([last_action[:, None].to(tokens.dtype), tokens], 1)
            column = torch.cat([column.new_full((1,), n - 1), column])
            time = torch.cat([rollouts.time - 1, time], 1)
        new = tokens.shape[1]
        if rollouts.taken + new > rollouts.tokens:
            raise ValueError("the rollouts' caches of %d tokens hold %d: no room for %d more"
                             % (rollouts.tokens, rollouts.taken, new))
        column = column.to(torch.int32).expand_as(time)
        pos = torch.stack([time, torch.zeros_like(time), column], 2)
        slots = rollouts.length + torch.arange(new, dtype=torch.int32, device=tokens.device)
        lo, hi = torch.zeros_like(slots), slots + 1

        def attend(i, block, q, k, v):
            keys, values = rollouts.caches[i]
            q = ops.norm_rotate_append(q, k, v, pos, self.freqs, self.sections, *block.weights(self.dtype), slots=slots,
                                       k_cache=keys, v_cache=values)
            return ops.range_attention_step(q, keys, values, lo, hi, cap=self.cap)

        logits = self._logits(tokens.contiguous(), attend, lambda x: x[:, -1])
        rollouts.taken += new
        rollouts.length += new
        rollouts.time += 1
        _, entropy, _, value, best = ops.token_log_probs(logits, scale=scale, top=top)
        return entropy, value, best
