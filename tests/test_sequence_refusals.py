"""What the operators between a batch of windows and a sequence model refuse, by name, before anything reaches the GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def test_on_the_host_arguments_are_named():
    from gear_amd import ops
    f = torch.zeros(2, 3, 4, 32)
    i = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="mask or done is needed"):
        ops.token_ranges()
    with pytest.raises(ValueError, match="mask and done must be"):
        ops.token_ranges(torch.zeros(3, dtype=torch.uint8))
    with pytest.raises(ValueError, match="mode must be 'causal', 'step' or 'document', got 'both'"):
        ops.token_ranges(i, mode="both")
    with pytest.raises(ValueError, match="tokens_per_step must be at least 1"):
        ops.token_ranges(i, tokens_per_step=0)
    with pytest.raises(ValueError, match="prefix must not be negative"):
        ops.token_ranges(i, prefix=-1)
    with pytest.raises(ValueError, match="grid must be"):
        ops.token_ranges(i, tokens_per_step=6, grid=(2, 2))
    with pytest.raises(TypeError, match="mask must have dtype torch.uint8 or torch.bool"):
        ops.token_ranges(i)
    with pytest.raises(ValueError, match="mask must live on the GPU"):
        ops.token_ranges(i.to(torch.uint8))
    with pytest.raises(TypeError, match="q must be a torch.Tensor"):
        ops.norm_rotate([1.0], f, i, f, [16])
    with pytest.raises(ValueError, match="q must live on the GPU"):
        ops.norm_rotate(f, f, i, f, [16])
    with pytest.raises(ValueError, match="q must be .batch, tokens, heads, head_dim."):
        ops.range_attention(f[0], f, f, i, i)
    with pytest.raises(ValueError, match="q must live on the GPU"):
        ops.range_attention_step(f.half(), f, f, i, i)


@pytest.mark.gpu
def test_norm_rotate_refuses():
    from gear_amd import ops
    q, k = torch.zeros(2, 3, 4, 32, device="cuda"), torch.zeros(2, 3, 1, 32, device="cuda")
    pos, freqs = torch.zeros(2, 3, 1, dtype=torch.int32, device="cuda"), torch.zeros(16, dtype=torch.float64, device="cuda")
    w = torch.ones(32, device="cuda")

    def refused(kind, match, q=q, k=k, pos=pos, freqs=freqs, sections=(16,), wq=w, wk=w, **more):
        with pytest.raises(kind, match=match):
            ops.norm_rotate(q, k, pos, freqs, sections, wq, wk, **more)

    refused(TypeError, "q must have dtype", q=q.double())
    refused(TypeError, "k must have dtype Float like q", k=k.half())
    refused(ValueError, "k must have shape", k=k[:1])
    refused(ValueError, "head_dim must be a multiple of 16", q=q[..., :24].contiguous(), k=k[..., :24].contiguous())
    refused(ValueError, "contiguous head_dim", q=q.transpose(2, 3))
    refused(ValueError, "multiples of 16 bytes", q=torch.zeros(2 * 3 * 4 * 32 + 1, device="cuda")[1:].view(2, 3, 4, 32))
    refused(ValueError, "more pairs than head_dim", sections=(10, 10))
    refused(ValueError, "sections must name 1 to 4 axes", sections=())
    refused(ValueError, "sections must be numbers of pairs", sections=(-1,))
    refused(ValueError, "pos must have shape .2, 3, 2.", sections=(8, 8))
    refused(TypeError, "pos must have dtype", pos=pos.long())
    refused(ValueError, "freqs must have shape .16.", freqs=freqs[:15])
    refused(TypeError, "freqs must have dtype torch.float64", freqs=freqs.float())
    refused(TypeError, "q_weight must have dtype torch.float32 or that of q", wq=w.half())
    refused(ValueError, "k_weight must have shape", wk=w[:16])
    refused(ValueError, "eps must be", eps=-1.0)
    refused(ValueError, "eps must be", eps=float("nan"))
    h = lambda x: x.half()  # noqa: E731
    refused(TypeError, "must have one dtype", q=h(q), k=h(k), wq=h(w))
    cache = torch.zeros(2, 9, 1, 32, device="cuda")
    slots = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for name, match in ((dict(slots=slots[:1]), "slots must have shape"), (dict(k_cache=cache[:, :, :, :16]), "k_cache must have shape"),
                        (dict(v_cache=cache[:, :5]), "v_cache must have shape")):
        with pytest.raises(ValueError, match=match):
            ops.norm_rotate_append(q, k, k, pos, freqs, (16,), w, w, **dict(dict(slots=slots, k_cache=cache, v_cache=cache), **name))
    with pytest.raises(ValueError, match="dq_out must have shape"):
        ops.norm_rotate_backward(k, k, q, k, pos, freqs, (16,), w, w)


@pytest.mark.gpu
def test_attention_refuses():
    from gear_amd import ops
    q, k = torch.zeros(2, 3, 4, 32, device="cuda").half(), torch.zeros(2, 5, 2, 32, device="cuda").half()
    lo = torch.zeros(2, 3, dtype=torch.int32, device="cuda")

    def refused(kind, match, q=q, k=k, v=k, lo=lo, hi=lo, **more):
        for call in (ops.range_attention, ops.range_attention_step):
            with pytest.raises(kind, match=match):
                call(q, k, v, lo, hi, **more)

    refused(TypeError, "q must have dtype torch.float16 or torch.bfloat16, got torch.float32", q=q.float(), k=k.float(), v=k.float())
    refused(TypeError, "must have dtype Half like q", k=k.bfloat16())
    refused(ValueError, "must have shape", v=k[:, :4])
    refused(ValueError, "heads of q must be a multiple", q=q[:, :, :3].contiguous())
    refused(ValueError, "head_dim must be a multiple of 16, at most 128", q=q.repeat(1, 1, 1, 5), k=k.repeat(1, 1, 1, 5), v=k.repeat(1, 1, 1, 5))
    refused(ValueError, "lo must have shape .2, 3.", lo=lo[:, :2].contiguous())
    refused(TypeError, "hi must have dtype", hi=lo.long())
    refused(ValueError, "scale must be", scale=0.0)
    refused(ValueError, "scale must be", scale=float("inf"))
    refused(ValueError, "cap must be", cap=-1.0)
    refused(ValueError, "slopes must have shape .4.", slopes=torch.zeros(2, device="cuda"))
    refused(TypeError, "slopes must have dtype", slopes=torch.zeros(4, device="cuda").half())
    out, lse = ops.range_attention(q, k, k, lo, lo)
    with pytest.raises(ValueError, match="dout must have shape"):
        ops.range_attention_backward(q[:, :2], q, k, k, out, lse, lo, lo)
    with pytest.raises(ValueError, match="lse must have shape"):
        ops.range_attention_backward(q, q, k, k, out, lse[:1], lo, lo)
    with pytest.raises(ValueError, match="out must be contiguous"):
        ops.range_attention_backward(q, q, k, k, out.transpose(1, 2), lse, lo, lo)


def test_codes_without_a_gpu():
    """The C entry points answer by codes before they touch the device."""
    from gear_amd import _cabi
    lib = _cabi.load()
    ranges = [1, 1, 1, 1, 1, 0, 0, 0, 0, None, None, None, None]
    assert lib.gear_hip_token_ranges(None, None, 0, 5, 1, 0, 0, 0, 0, None, None, None, None) == 0
    assert lib.gear_hip_token_ranges(None, None, *ranges[2:]) == -1
    assert lib.gear_hip_token_ranges(None, None, 1, 1, 1, 3, 0, 0, 0, None, None, None, None) == -1
    assert lib.gear_hip_token_ranges(None, None, 1, 1 << 30, 4, 0, 0, 0, 0, None, None, None, None) == -3
    assert lib.gear_hip_token_ranges(None, None, 1, 1, 6, 0, 0, 2, 2, None, None, None, None) == -1

    norm = _cabi.NormRotateDesc(batch=0, tokens=3, q_heads=1, k_heads=1, head_dim=32, axes=1, eps=0.0)
    byref = ctypes.byref
    assert lib.gear_hip_norm_rotate(None, None, None, None) == -1
    assert lib.gear_hip_norm_rotate(byref(norm), None, None, None) == 0
    norm.batch = 1
    assert lib.gear_hip_norm_rotate(byref(norm), None, None, None) == -1
    norm.head_dim = 272
    assert lib.gear_hip_norm_rotate(byref(norm), None, None, None) == -3
    norm.head_dim = 40
    assert lib.gear_hip_norm_rotate(byref(norm), None, None, None) == -1
    norm.head_dim, norm.sections[0] = 32, 17
    assert lib.gear_hip_norm_rotate(byref(norm), None, None, None) == -1
    assert lib.gear_hip_norm_rotate_backward_workspace_bytes(128) > 0

    att = _cabi.AttentionDesc(batch=0, queries=3, keys=3, heads=2, kv_heads=1, head_dim=32, dtype=1, scale=1.0)
    assert lib.gear_hip_attention(byref(att), None, None, None) == 0
    att.batch = 1
    assert lib.gear_hip_attention(byref(att), None, None, None) == -1
    assert lib.gear_hip_attention(None, None, None, None) == -1
    for name, value, code in (("scale", 0.0, -1), ("scale", float("nan"), -1), ("cap", -1.0, -1), ("kv_heads", 3, -1), ("dtype", 0, -1),
                              ("head_dim", 144, -3), ("queries", 1 << 30, -3), ("head_dim", 20, -1)):
        bad = _cabi.AttentionDesc(batch=1, queries=3, keys=3, heads=2, kv_heads=1, head_dim=32, dtype=1, scale=1.0)
        setattr(bad, name, value)
        assert lib.gear_hip_attention(byref(bad), None, None, None) == code, name
        assert lib.gear_hip_attention_step(byref(bad), None, None, 0, None) == code, name
    # sizes of scratch: by host arithmetic
    assert lib.gear_hip_attention_backward_workspace_bytes(2, 100, 4) >= 4 * 2 * 100 * 4 + 2 * 4 * 16
    assert lib.gear_hip_attention_step_workspace_bytes(1, 1, 100, 8, 8, 64) == 0
    assert lib.gear_hip_attention_step_workspace_bytes(1, 1, 100_000, 8, 1, 64) > 0


def test_scales_and_caps_that_32_bits_do_not_hold():
    """By code before the device is touched: a scale and a cap below 1e30, and a scale below 1e30 times the cap."""
    from gear_amd import _cabi
    lib = _cabi.load()
    for scale, cap, code in ((1e30, 0.0, -1), (1.0, 1e30, -1), (1.0, 1e-30, -1), (1e10, 1e-25, -1), (1.0, 1e-29, 0), (1.0, 1e29, 0),
                             (1e29, 1e29, 0)):
        att = _cabi.AttentionDesc(batch=0, queries=3, keys=3, heads=2, kv_heads=1, head_dim=32, dtype=1, scale=scale, cap=cap)
        assert lib.gear_hip_attention(ctypes.byref(att), None, None, None) == code, (scale, cap)


@pytest.mark.gpu
def test_attention_refuses_caps_and_scales_by_name():
    from gear_amd import ops
    q, lo = torch.zeros(2, 3, 4, 32, device="cuda").half(), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for call in (ops.range_attention, ops.range_attention_step):
        for cap in (1e30, 1e300, 1e-31, 1e-300):
            with pytest.raises(ValueError, match="cap must be"):
                call(q, q, q, lo, lo, cap=cap)
        with pytest.raises(ValueError, match="scale must be"):
            call(q, q, q, lo, lo, scale=1e30)
        with pytest.raises(ValueError, match="scale must be"):
            call(q, q, q, lo, lo, scale=1e-300)


def test_launches_that_cannot_be():
    """2^32 work items and more are refused by code, before the device is touched (the pointers are no memory)."""
    from gear_amd import _cabi
    lib, none = _cabi.load(), ctypes.c_void_p(256)

    def attention(**sizes):
        return _cabi.AttentionDesc(**dict(dict(q=256, k=256, v=256, lo=256, hi=256, batch=1, queries=1, keys=1, heads=1, kv_heads=1,
                                               head_dim=128, dtype=1, scale=1.0), **sizes))

    strides = (ctypes.c_int64 * 3)(0, 0, 0)
    forward = lambda d: lib.gear_hip_attention(ctypes.byref(d), none, none, None)  # noqa: E731
    backward = lambda d: lib.gear_hip_attention_backward(  # noqa: E731
        ctypes.byref(d), none, strides, none, none, none, none, none, none, 1 << 60, None)
    step = lambda d: lib.gear_hip_attention_step(ctypes.byref(d), none, none, 1 << 60, None)  # noqa: E731
    most = 1 << 20
    assert forward(attention(batch=most, heads=64, kv_heads=64)) == -3  # one wave each
    assert forward(attention(batch=most, heads=16, kv_heads=16, queries=128)) == -3  # four
    assert forward(attention(batch=1, heads=2, kv_heads=1, queries=(1 << 30) - 1)) == -3
    assert backward(attention(batch=most, heads=64, kv_heads=64, head_dim=64)) == -3  # in one launch
    assert backward(attention(batch=most, heads=64, kv_heads=64, queries=200, keys=0)) == -3  # in two
    assert backward(attention(batch=most, heads=16, kv_heads=16)) == -3  # the keys' side: four waves always
    assert step(attention(batch=most, heads=16, kv_heads=16)) == -3
    assert step(attention(batch=1, queries=1 << 20, heads=1 << 15, kv_heads=1 << 10)) == -3
