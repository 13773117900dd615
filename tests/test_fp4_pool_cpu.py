"""KVPages, FP4KVPool and the block's calls on them, without a GPU: what they refuse, and where and with what they launch."""
import pytest
import torch

from goml_b200 import nn


@pytest.mark.parametrize("scale", [float("inf"), 1e39, 7.7e35, 1e-46, 0.0, -1.0, float("nan")])
def test_scales_that_the_cache_cannot_have(scale):
    # 448 of a scale have to be a number of 32 bits, and the scale itself one above zero
    pages = nn.KVPages(2, 8, 64, 3, device="cpu")
    for name in ("k_scale", "v_scale"):
        with pytest.raises(ValueError, match="FP4KVPool"):
            nn.FP4KVPool(pages, 2, 64, **{name: scale})


@pytest.mark.parametrize("scale", [2.0 ** -149, 1e-40, 1 / 32, 7.5e35])
def test_scales_that_it_can(scale):
    pool = nn.FP4KVPool(nn.KVPages(2, 8, 64, 3, device="cpu"), 2, 64, k_scale=scale, v_scale=scale)
    assert (pool.scales > 0).all() and torch.isfinite(448 * pool.scales).all()
