"""What of the sequence model needs no GPU."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("parameters", [torch.float16, torch.bfloat16, torch.float64])
def test_casts_leave_the_frequencies(parameters):
    from gear_amd.sequence import WindowModel
    model = WindowModel(5, 3, width=64, heads=2, kv_heads=1)
    want = model.freqs.clone()
    for cast in (lambda m: m.to(parameters), lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.float(), lambda m: m.double()):
        assert cast(model) is model
        assert model.freqs.dtype == torch.float64 and torch.equal(model.freqs, want)
    assert "freqs" in dict(model.named_buffers()) and "freqs" not in model.state_dict()
    assert all(p.dtype == torch.float64 for p in model.parameters())


def test_a_model_without_memory_gets_its_frequencies_with_it():
    from gear_amd.sequence import WindowModel
    want = WindowModel(5, 3, width=64, heads=2, kv_heads=1).freqs
    model = WindowModel(5, 3, width=64, heads=2, kv_heads=1).to("meta")
    assert model.freqs.is_meta and model.freqs.dtype == torch.float64
    model = model.to_empty(device="cpu")
    assert torch.equal(model.freqs, want)
