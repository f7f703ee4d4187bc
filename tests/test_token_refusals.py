"""What the operators of token models refuse, by name, before anything reaches the GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def test_on_the_host_arguments_are_named():
    from gear_amd import ops
    f, i = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError, match="tokens must be a torch.Tensor"):
        ops.embed_tokens([1], f)
    with pytest.raises(TypeError, match="tokens must have dtype torch.int64 or torch.int32, got torch.int16"):
        ops.embed_tokens(i.short(), f)
    with pytest.raises(ValueError, match="tokens must live on the GPU"):
        ops.embed_tokens(i, f)
    with pytest.raises(ValueError, match="dout must live on the GPU"):
        ops.embed_tokens_backward(f, i, 3)
    with pytest.raises(TypeError, match="x must have dtype torch.float32, torch.float16 or torch.bfloat16, got torch.float64"):
        ops.layer_norm(f.double())
    with pytest.raises(ValueError, match="x must live on the GPU"):
        ops.layer_norm(f)
    with pytest.raises(ValueError, match="logits must live on the GPU"):
        ops.token_log_probs(f)
    with pytest.raises(TypeError, match="logits must be a torch.Tensor"):
        ops.distill(None, i, f)
    from gear_amd.sequence import TokenModel
    with pytest.raises(ValueError, match="two tokens at least"):
        TokenModel(10, 1)


@pytest.mark.gpu
def test_embed_refuses():
    from gear_amd import ops
    table, tokens = torch.zeros(9, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    dout = torch.zeros(4, 16, device="cuda")
    for kind, match, call in (
            (ValueError, "table must be .vocab, width.", lambda: ops.embed_tokens(tokens, table[0])),
            (ValueError, "table must have at least one element a row", lambda: ops.embed_tokens(tokens, table[:, :0])),
            (TypeError, "table must have dtype", lambda: ops.embed_tokens(tokens, table.double())),
            (ValueError, "table must have contiguous elements", lambda: ops.embed_tokens(tokens, table.t())),
            (ValueError, "table must live on the GPU", lambda: ops.embed_tokens(tokens, table.cpu())),
            (ValueError, "tokens must be contiguous", lambda: ops.embed_tokens(tokens[::2], table)),
            (ValueError, "scale must be a finite number", lambda: ops.embed_tokens(tokens, table, scale=float("inf"))),
            (ValueError, "tokens must have shape .4., got .2.", lambda: ops.embed_tokens_backward(dout, tokens[:2], 9)),
            (ValueError, "vocab must be", lambda: ops.embed_tokens_backward(dout, tokens, -1)),
            (ValueError, "vocab must be", lambda: ops.embed_tokens_backward(dout, tokens, 2 ** 31)),
            (ValueError, "rows at one stride", lambda: ops.embed_tokens_backward(torch.zeros(2, 4, 16, device="cuda").transpose(0, 1),
                                                                                 torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 9))):
        with pytest.raises(kind, match=match):
            call()


@pytest.mark.gpu
def test_layer_norm_refuses():
    from gear_amd import ops
    x, w = torch.zeros(4, 16, device="cuda"), torch.zeros(16, device="cuda")
    for kind, match, call in (
            (ValueError, "at most 16384 elements", lambda: ops.layer_norm(torch.zeros(1, 16385, device="cuda"))),
            (ValueError, "x must have at least one dimension", lambda: ops.layer_norm(x[0, 0])),
            (TypeError, "weight must have dtype torch.float32 or that of the rows", lambda: ops.layer_norm(x, w.half())),
            (TypeError, "weight and bias must have one dtype", lambda: ops.layer_norm(x.half(), w, w.half())),
            (ValueError, "bias must have shape .16., got .8.", lambda: ops.layer_norm(x, w, w[:8])),
            (ValueError, "weight must be contiguous", lambda: ops.layer_norm(x, torch.zeros(32, device="cuda")[::2])),
            (ValueError, "eps must be", lambda: ops.layer_norm(x, eps=-1.0)),
            (ValueError, "eps must be", lambda: ops.layer_norm(x, eps=float("nan"))),
            (ValueError, "residual must have shape", lambda: ops.layer_norm(x, residual=x[:2])),
            (TypeError, "residual must have the dtype of x", lambda: ops.layer_norm(x, residual=x.half())),
            (ValueError, "residual must have contiguous elements", lambda: ops.layer_norm(x, residual=torch.zeros(16, 4, device="cuda").t())),
            (ValueError, "dy must have shape", lambda: ops.layer_norm_backward(x[:, :8], x)),
            (ValueError, "dsum must live on the GPU", lambda: ops.layer_norm_backward(x, x, dsum=x.cpu()))):
        with pytest.raises(kind, match=match):
            call()


@pytest.mark.gpu
def test_logits_refuse():
    from gear_amd import ops
    x, tokens, f = torch.zeros(4, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, device="cuda")
    best, t = torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.zeros(4, 2, device="cuda")
    for kind, match, call in (
            (ValueError, "at most 2.20 tokens a row", lambda: ops.token_log_probs(torch.zeros(1, 2 ** 20 + 1, device="cuda"))),
            (ValueError, "logits must have at least one element a row", lambda: ops.token_log_probs(x[:, :0])),
            (ValueError, "scale must be a number above 0", lambda: ops.token_log_probs(x, scale=0.0)),
            (ValueError, "scale must be a number above 0", lambda: ops.token_log_probs(x, scale=float("nan"))),
            (ValueError, "top must be", lambda: ops.token_log_probs(x, top=17)),
            (ValueError, "top must be", lambda: ops.token_log_probs(torch.zeros(1, 99, device="cuda"), top=65)),
            (ValueError, "top must be", lambda: ops.token_log_probs(x, top=-1)),
            (ValueError, "tokens must have shape .4., got .3.", lambda: ops.token_log_probs(x, tokens[:3])),
            (TypeError, "tokens must have dtype", lambda: ops.token_log_probs(x, f)),
            (ValueError, "logits must have contiguous elements", lambda: ops.token_log_probs(x.t())),
            (ValueError, "lse is needed", lambda: ops.token_log_probs_backward(f, None, x, tokens, None, None)),
            (ValueError, "dlog_probs needs the tokens", lambda: ops.token_log_probs_backward(f, None, x, None, f, None)),
            (ValueError, "dentropy needs the entropy", lambda: ops.token_log_probs_backward(None, f, x, None, f, None)),
            (TypeError, "dlog_probs must have dtype torch.float32", lambda: ops.token_log_probs_backward(f.half(), None, x, tokens, f, f)),
            (ValueError, "lse must have shape", lambda: ops.token_log_probs_backward(f, None, x, tokens, f[:2], f)),
            (ValueError, "1 to 64 tokens", lambda: ops.distill(x, best[:, :0], t[:, :0])),
            (ValueError, "1 to 64 tokens", lambda: ops.distill(x, best.repeat(1, 33), t.repeat(1, 33))),
            (ValueError, "top_tokens must have shape", lambda: ops.distill(x, best[:2], t[:2])),
            (ValueError, "top_logits must have shape", lambda: ops.distill(x, best, t[:, :1].contiguous())),
            (TypeError, "top_logits must have dtype torch.float32", lambda: ops.distill(x, best, t.half())),
            (ValueError, "top_logits is needed", lambda: ops.distill(x, best, None)),
            (ValueError, "top_tokens must be contiguous", lambda: ops.distill(x, best.t().contiguous().t(), t)),
            (ValueError, "dloss must have shape", lambda: ops.distill_backward(f[:2], x, best, t, f)),
            (ValueError, "dloss and lse are needed", lambda: ops.distill_backward(f, x, best, t, None))):
        with pytest.raises(kind, match=match):
            call()


def test_codes_without_a_gpu():
    """The C entry points answer by codes before they touch the device."""
    from gear_amd import _cabi
    lib = _cabi.load()
    f = ctypes.c_float
    some = 4096  # an address that is never read
    embed = lib.gear_hip_embed
    assert embed(None, 1, 0, None, 0, 5, 8, 0, f(1), None, None) == 0
    assert embed(None, 1, 3, None, 0, 5, 8, 0, f(1), None, None) == -1
    assert embed(some, 1, -1, some, 8, 5, 8, 0, f(1), some, None) == -1
    assert embed(some, 1, 1, some, 8, 5, 0, 0, f(1), some, None) == -1
    assert embed(some, 1, 1, some, 8, 5, 8, 3, f(1), some, None) == -1
    assert embed(some, 1, 1, some, 8, 5, 8, 0, f(float("nan")), some, None) == -1
    assert embed(some, 1, 1 << 31, some, 8, 5, 8, 0, f(1), some, None) == -3
    assert embed(some, 1, 1, some, 8, 1 << 31, 8, 0, f(1), some, None) == -3
    assert embed(some, 1, 1, some, 8, 5, (1 << 20) + 1, 0, f(1), some, None) == -3
    assert embed(some + 4, 1, 1, some, 8, 5, 8, 0, f(1), some, None) == -4
    assert embed(some, 0, 1, some + 1, 8, 5, 8, 1, f(1), some, None) == -4
    back, need = lib.gear_hip_embed_backward, lib.gear_hip_embed_backward_workspace_bytes
    assert need(0, 8) == 0 and need(1, 8) > 0 and need(1 << 31, 8) == 0
    assert back(some, 8, some, 1, 3, 5, 8, 0, f(1), some, None, 0, None) == -2
    assert back(some, 8, some, 1, 3, 5, 8, 0, f(1), some, some, need(3, 8) - 1, None) == -2
    assert back(some, 8, some, 1, 3, 5, 8, 0, f(1), some, some + 8, need(3, 8), None) == -4
    assert back(None, 0, None, 1, 3, 0, 8, 0, f(1), None, None, 0, None) == 0
    assert back(None, 0, some, 1, 3, 5, 8, 0, f(1), some, None, 0, None) == -1
    # more work items than a launch has
    assert back(some, 8, some, 1, (1 << 31) - 1, 5, 1 << 20, 0, f(1), some, some, 1 << 62, None) == -3

    def norm(**over):
        d = _cabi.LayerNormDesc(x=some, x_stride=8, rows=3, width=8, dtype=0, weight_f32=1, eps=1e-5)
        for k, v in over.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    forward, backward = lib.gear_hip_layer_norm, lib.gear_hip_layer_norm_backward
    assert forward(None, some, None, None) == -1
    assert forward(norm(rows=0), None, None, None) == 0
    assert forward(norm(rows=-1), some, None, None) == -1
    assert forward(norm(width=0), some, None, None) == -1
    assert forward(norm(width=16385), some, None, None) == -3
    assert forward(norm(eps=-1.0), some, None, None) == -1
    assert forward(norm(dtype=5), some, None, None) == -1
    assert forward(norm(x=None), some, None, None) == -1
    assert forward(norm(), None, None, None) == -1
    assert forward(norm(residual=some), some, None, None) == -1
    assert forward(norm(), some, some, None) == -1
    assert forward(norm(x=some + 2), some, None, None) == -4
    assert forward(norm(weight=some + 2), some, None, None) == -4
    assert lib.gear_hip_layer_norm_backward_workspace_bytes(3, 16385) == 0
    assert backward(norm(), some, 8, None, 0, some, some, None, None, 0, None) == -2
    assert backward(norm(), None, 8, None, 0, some, None, None, None, 0, None) == -1
    assert backward(norm(), some, 8, None, 0, None, None, None, None, 0, None) == -1
    assert backward(norm(rows=0), None, 0, None, 0, None, None, None, None, 0, None) == 0

    def rows(**over):
        d = _cabi.LogitsDesc(logits=some, row_stride=99000, rows=3, vocab=99000, dtype=0, scale=1.0)
        for k, v in over.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    log_probs = lib.gear_hip_token_log_probs
    need = lib.gear_hip_token_log_probs_workspace_bytes
    outs = (some, some, some)
    assert need(3, 99000, 0) > 0 and need(3, 99000, 64) > need(3, 99000, 0) and need(100000, 9000, 64) == 0
    assert need(3, 1 << 21, 0) == 0 and need(3, 99000, 65) == 0 and need(0, 9000, 0) == 0
    assert log_probs(None, None, 1, 0, None, some, some, None, None, None, 0, None) == -1
    assert log_probs(rows(rows=0), None, 1, 0, None, None, None, None, None, None, 0, None) == 0
    assert log_probs(rows(vocab=0), None, 1, 0, None, some, some, None, None, None, 0, None) == -1
    assert log_probs(rows(vocab=(1 << 20) + 1), None, 1, 0, None, some, some, None, None, None, 0, None) == -3
    for scale in (0.0, -1.0, 1e30, float("nan")):
        assert log_probs(rows(scale=scale), None, 1, 0, None, some, some, None, None, None, 0, None) == -1
    assert log_probs(rows(), some, 1, 0, None, some, some, None, None, some, 1 << 30, None) == -1
    assert log_probs(rows(), None, 1, 0, *outs, None, None, some, 1 << 30, None) == -1
    assert log_probs(rows(), some, 1, 2, *outs, None, None, some, 1 << 30, None) == -1
    assert log_probs(rows(), some, 1, 99001, *outs, some, some, some, 1 << 30, None) == -1
    assert log_probs(rows(), some, 1, 65, *outs, some, some, some, 1 << 30, None) == -3
    assert log_probs(rows(), some, 1, 2, *outs, some, some, None, 0, None) == -2
    assert log_probs(rows(), some, 1, 2, *outs, some, some, some, need(3, 99000, 2) - 1, None) == -2
    assert log_probs(rows(), some, 1, 2, *outs, some, some, some + 128, 1 << 30, None) == -4
    assert log_probs(rows(logits=some + 2), some, 1, 0, *outs, None, None, some, 1 << 30, None) == -4
    grad = lib.gear_hip_token_log_probs_backward
    assert grad(rows(), some, None, None, 1, some, None, some, None) == -1
    assert grad(rows(), None, some, None, 1, some, None, some, None) == -1
    assert grad(rows(), some, some, some, 1, None, some, some, None) == -1
    assert grad(rows(rows=0), None, None, None, 1, None, None, None, None) == 0
    assert grad(rows(rows=(1 << 31) - 1), None, some, None, 1, some, some, some, None) == -3
    assert lib.gear_hip_distill(rows(), some, 1, some, 0, some, some, some, 1 << 30, None) == -1
    assert lib.gear_hip_distill(rows(), some, 1, some, 65, some, some, some, 1 << 30, None) == -3
    assert lib.gear_hip_distill(rows(), some, 1, some, 8, some, some, None, 0, None) == -2
    assert lib.gear_hip_distill(rows(), some, 1, None, 8, some, some, some, 1 << 30, None) == -1
    assert lib.gear_hip_distill_backward(rows(), None, some, 1, some, 8, some, some, None) == -1
    assert lib.gear_hip_distill_backward(rows(), some, some + 4, 1, some, 8, some, some, None) == -4
