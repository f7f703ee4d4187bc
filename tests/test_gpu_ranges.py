"""Ranges of keys and positions of windows against a step-by-step statement in numpy: whole numbers, equal."""
import numpy as np
import pytest

from conftest import announce
from sequence_reference import token_ranges

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

MODES = [("causal", 0), ("step", 0), ("document", 0), ("causal", 3), ("step", 1), ("document", 5), ("causal", 1000)]


def _check(mask, done, tokens, mode, prefix, grid=None, as_bool=False):
    from gear_amd import ops
    kind = np.bool_ if as_bool else np.uint8
    up = lambda x: None if x is None else torch.from_numpy(x.astype(kind)).cuda()  # noqa: E731
    got = ops.token_ranges(up(mask), up(done), tokens_per_step=tokens, mode=mode, prefix=prefix, grid=grid)
    shape = (mask if mask is not None else done).shape
    want = token_ranges(np.ones(shape, int) if mask is None else mask, np.zeros(shape, int) if done is None else done,
                        tokens, mode, prefix, grid)
    for name, g, w in zip(("lo", "hi", "pos"), got, want):
        assert g.dtype == torch.int32 and g.shape == w.shape, name
        assert np.array_equal(g.cpu().numpy(), w), name


@pytest.mark.parametrize("steps", [1, 2, 20, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("tokens", [1, 3])
def test_windows(steps, tokens):
    rng = np.random.default_rng(steps * 10 + tokens)
    for ends in (0.0, 0.1, 0.9):
        mask = np.zeros((11, steps), np.uint8)
        for b in range(11):  # head padding, tail padding, holes, empty, full
            n = int(rng.integers(0, steps + 1))
            if b == 0:
                mask[b] = 1
            elif b % 3 == 0:
                mask[b, :n] = 200
            elif b % 3 == 1:
                mask[b, steps - n:] = 1
            else:
                mask[b] = rng.random(steps) < 0.7
        mask[5] = 0
        done = (rng.random((11, steps)) < ends).astype(np.uint8) * 255
        for mode, prefix in MODES:
            announce("ranges steps=%d tokens=%d ends=%g %s prefix=%d" % (steps, tokens, ends, mode, prefix))
            _check(mask, done, tokens, mode, prefix)


def test_documents_far_longer_than_a_wave():
    """Documents that begin thousands of steps before and end thousands of steps behind a wave's steps."""
    rng = np.random.default_rng(3)
    mask, done = np.ones((4, 5000), np.uint8), np.zeros((4, 5000), np.uint8)
    mask[1, :17] = 0
    mask[1, 4990:] = 0
    done[2, [0, 63, 64, 1087, 1088, 4999]] = 1
    mask[3] = rng.random(5000) < 0.999
    done[3] = rng.random(5000) < 0.001
    for mode, prefix in MODES:
        announce("long documents %s prefix=%d" % (mode, prefix))
        _check(mask, done, 1, mode, prefix)


def test_grids_missing_arguments_and_bool():
    rng = np.random.default_rng(4)
    mask, done = (rng.random((3, 70)) < 0.9).astype(np.uint8), (rng.random((3, 70)) < 0.05).astype(np.uint8)
    announce("grids")
    for grid in ((7, 7), (1, 5), (6, 1), (2, 3)):
        _check(mask, done, grid[0] * grid[1], "step", 2, grid)
    _check(mask, done, 2, "document", 0, as_bool=True)
    _check(None, done, 2, "causal", 0)
    _check(mask, None, 2, "document", 0)


def test_nothing_to_do_and_a_table_slice():
    from gear_amd import ops
    announce("empty batches, a bool mask made on the GPU")
    for shape in ((0, 5), (5, 0)):
        lo, hi, pos = ops.token_ranges(torch.zeros(shape, dtype=torch.uint8, device="cuda"), tokens_per_step=2)
        assert lo.shape == hi.shape == (shape[0], shape[1] * 2) and pos.shape == (shape[0], shape[1] * 2, 1)
    lo, hi, _ = ops.token_ranges(torch.ones(2, 4, device="cuda") > 0)
    assert hi.tolist() == [[1, 2, 3, 4]] * 2 and not lo.any()


def test_windows_beyond_one_launch():
    """A launch has less than 2^32 work items, a wave a window: 2^26 windows and some are two."""
    from gear_amd import ops
    announce("2^26 + 5 windows of one step")
    mask = (torch.arange((1 << 26) + 5, device="cuda") % 7 != 3).to(torch.uint8)[:, None].contiguous()
    lo, hi, pos = ops.token_ranges(mask)
    assert torch.equal(hi, mask.int()) and not lo.any() and not pos.any()
    announce("2^25 + 3 windows of 65 steps")
    mask = torch.ones((1 << 25) + 3, 65, dtype=torch.bool, device="cuda")
    mask[-1, 40] = False
    lo, hi, pos = ops.token_ranges(mask)
    want = ops.token_ranges(mask[-2:].contiguous())
    assert all(torch.equal(a[-2:], b) for a, b in zip((lo, hi, pos), want))
    at = torch.arange(65, dtype=torch.int32, device="cuda")
    assert bool((hi[:-1] == at + 1).all()) and not lo[:-1].any() and bool((pos[:-1, :, 0] == at).all())
