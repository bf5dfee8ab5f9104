"""What the paged cache's calls take and refuse beside plain arguments (CPU)."""

import pytest
import torch

from foveated_kv_amd import Rope, paged
from test_paged import SCALINGS


@pytest.mark.parametrize("scaling", SCALINGS)
def test_rope_under_another_default_device(scaling):
    """The frequencies are host memory whatever torch's default device is."""
    want = Rope(64, scaling=scaling, max_positions=40, device="cpu").table
    with torch.device("meta"):
        inv, _ = paged._frequencies(64, 10000.0, scaling)
        assert inv.device.type == "cpu" and inv.is_contiguous()
        got = Rope(64, scaling=scaling, max_positions=40, device="cpu").table
    assert got.device.type == "cpu" and torch.equal(got, want)
