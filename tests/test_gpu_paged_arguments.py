"""What the paged cache's calls take and refuse beside plain arguments (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.calls()
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def test_a_cuda_default_device(paged):
    """A program whose new tensors are the GPU's: the same table, cache and
    results."""
    def run():
        rope = paged.Rope(64, rot_dim=32, scaling={"kind": "ntk", "factor": 2.0}, max_positions=100)
        cache = paged.PagedKVCache(1, 2, 64, n_pages=8, max_seqs=2, max_tokens=64, page_size=16, rope=rope)
        g = torch.Generator(device="cpu").manual_seed(0)
        k, v, q = (torch.randn(2, h, n, 64, generator=g, device="cpu").half().cuda() for h, n in ((2, 5), (2, 5), (4, 5)))
        cache.extend([5, 3])
        cache.write(0, k, v)
        cache.extend(1)
        qr = cache.write(0, k[:, :, :1], v[:, :, :1], q=q[:, :, :1])
        return [rope.table, qr, cache.attend(0, qr), *cache.read(0)]

    want = run()
    with torch.device("cuda"):
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
