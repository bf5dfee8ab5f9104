"""Rotations and writes of more rows than the small calls' kernels take: the
bits that the same rows give in calls of fewer, which the other tests hold to
the 64-bit restatements."""

import pytest
import torch

pytestmark = pytest.mark.gpu

FEW = 16384  # rows up to which a lane takes one at a time


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.load()
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def _equal(a, b, what):
    a, b = (t.view(torch.uint8) for t in (a.contiguous(), b.contiguous()))
    assert torch.equal(a, b), f"{what}: {int((a != b).sum())} bytes differ"


def _pieces(L, rows):
    """Runs of an odd number of the L tokens of `rows` rows, few rows each."""
    step = min(L // 2, FEW // rows) // 2 * 2 - 1
    return [(a, min(a + step, L)) for a in range(0, L, step)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (128, 128, True), (64, 16, False), (64, 32, True),
                                               (80, 48, False), (256, 256, False), (512, 64, True)])
@pytest.mark.parametrize("H", [1, 5, 13, 66])
def test_rotary(paged, dtype, D, rot, interleaved, H):
    print("rotary", dtype, D, rot, interleaved, H, flush=True)
    B = 3
    L = FEW // (B * H) + 101
    rope = paged.Rope(D, rot_dim=rot, interleaved=interleaved, max_positions=L + 20)
    x = _randn(H, B, L, H, D).to("cuda", dtype).transpose(1, 2)
    start = torch.tensor([0, 37, 11], dtype=torch.int32, device="cuda")  # (the second one's last are outside)
    assert B * H * L > FEW
    got = rope(x, start)
    for a, b in _pieces(L, B * H):
        _equal(got[:, :, a:b], rope(x[:, :, a:b], start + a), f"tokens {a} to {b}")
    y = x.clone()
    assert rope(y, start, out=y) is y
    _equal(y, got, "in place")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot,interleaved", [(128, 0, False), (128, 128, False), (64, 64, True), (64, 16, False),
                                               (128, 32, True)])
@pytest.mark.parametrize("H,Hq", [(3, 7), (1, 18), (5, 0), (8, 8)])
def test_write(paged, dtype, D, rot, interleaved, H, Hq):
    print("write", dtype, D, rot, interleaved, H, Hq, flush=True)
    B, page = 3, 32
    L = FEW // (B * (2 * H + Hq)) + 131
    P = -(-(L + 40) // page)
    k, v, q = (_randn(s + H, B, n, L, D).to("cuda", dtype) for s, n in ((1, H), (2, H), (3, max(Hq, 1))))
    k[..., 3] *= 8.0
    table = torch.randperm(B * P, generator=torch.Generator().manual_seed(4)).to("cuda", torch.int32).view(B, P)
    table[2, 5] = -1  # (tokens of a page outside the pool are not stored)
    rope = paged.Rope(D, rot_dim=rot, interleaved=interleaved, max_positions=L + 50) if rot else None
    start = torch.tensor([0, 37, 11], dtype=torch.int32, device="cuda")
    n_new = torch.tensor([L, L - 13, 0 if H == 5 else L // 2], dtype=torch.int32, device="cuda")
    assert B * (2 * H + Hq) * L > FEW
    for fmt in ("fp16", "bf16", "fp8", "fp8_int4"):
        for lens in (None, n_new):
            whole, parts = (paged.PagedLayer(B * P, H, D, page, fmt) for _ in range(2))
            got = whole.write(k, v, table, start, n_new=lens, q=q if Hq else None, rope=rope)
            for a, b in _pieces(L, B * (2 * H + Hq)):
                r = parts.write(k[:, :, a:b], v[:, :, a:b], table, start + a, n_new=None if lens is None else lens - a,
                                q=q[:, :, a:b] if Hq else None, rope=rope)
                if Hq:
                    _equal(got[:, :, a:b], r, f"{fmt}, queries {a} to {b}")
            for name in ("k", "v", "k_exp", "v_scale"):
                if getattr(whole, name) is not None:
                    _equal(getattr(whole, name), getattr(parts, name), f"{fmt}, {name}")
