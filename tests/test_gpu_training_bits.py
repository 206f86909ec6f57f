"""A deterministic training gives the same bits again, whatever the GPU's memory held before: nothing that a step reads is
left unwritten, and no step depends on the order in which work happens to arrive."""
import hashlib

import pytest
import torch

import density_slices_util as D

pytestmark = pytest.mark.gpu


def bits(path, background, steps):
    """The whole state (weights, moments, density grid, counters) after each of `steps`, and what the step reported."""
    import pyngp as ngp
    tb = D.new_testbed(ngp, "test2", "base.json", 1337, random_bg_color=background)
    tb.deterministic = True
    out = []
    for n in steps:
        D.train_to(tb, n)
        tb.save_snapshot(path, True)
        with open(path, "rb") as f:
            out.append((n, hashlib.sha256(f.read()).hexdigest(), tb.last_train_stats()["n_rays"], tb.last_train_stats()["loss"]))
    return out


@pytest.mark.parametrize("background", [True, False])
def test_training_gives_the_same_bits_whatever_the_memory_held(tmp_path, background):
    steps = (1, 20, 300, 800)
    first = bits(str(tmp_path / "a.msgpack"), background, steps)
    for fill in (float("nan"), -1.0):
        held = [torch.full((1 << 28,), fill, device="cuda") for _ in range(32)]  # 32 GiB, given back to the driver
        torch.cuda.synchronize()
        del held
        torch.cuda.empty_cache()
        assert bits(str(tmp_path / "b.msgpack"), background, steps) == first
