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


class _Recorded:
    """A cache whose pages are handed out and whose layers only note calls."""

    rope, layers = None, [None]

    def __init__(self, fails=False):
        self.pages, self.done, self.fails = paged.PageTable(8, 16, 2, 64, device="cpu"), [], fails

    def write(self, *args, **kw):
        self.done.append("write")
        if self.fails:
            raise RuntimeError("no write")

    def read(self, layer, seqs, dtype):
        self.done.append("read")
        return "k", "v"


def test_chunks_at_different_beginnings():
    """Whether there is something to read back is a matter of every sequence's
    beginning, which the host knows."""
    from foveated_kv_amd import generate

    cache, kv = _Recorded(), torch.zeros(2, 1, 5, 64)
    w, = generate.install_paged_attention(cache)
    try:
        cache.pages.extend(5)
        assert w.offset == 0 and w.update_and_fetch(kv, kv) == (kv, kv) and cache.done == ["write"]
        torch.nn.functional.scaled_dot_product_attention(kv, kv, kv)
        cache.pages.free(1)
        cache.pages.extend(5)
        assert w.offset.tolist() == [5, 0]
        assert w.update_and_fetch(kv, kv) == ("k", "v") and cache.done == ["write", "write", "read"]
        torch.nn.functional.scaled_dot_product_attention(kv, kv, kv)
    finally:
        generate.uninstall_paged_attention()


def test_a_failed_update_leaves_nothing_pending():
    from foveated_kv_amd import generate

    cache, kv = _Recorded(fails=True), torch.zeros(2, 1, 5, 64)
    w, = generate.install_paged_attention(cache)
    try:
        for _ in range(2):
            with pytest.raises(RuntimeError, match="no write"):
                w.update_and_fetch(kv, kv)
        torch.nn.functional.scaled_dot_product_attention(kv[:, :, :2], kv, kv)  # (another attention)
    finally:
        generate.uninstall_paged_attention()


def test_a_forward_tangent_is_refused():
    from torch.autograd import forward_ad

    x = torch.zeros(1, 2, 3, 64)
    with forward_ad.dual_level():
        paged._on(-1, "x", x)
        with pytest.raises(RuntimeError, match="tangent"):
            paged._on(-1, "x", forward_ad.make_dual(x, torch.ones_like(x)))
