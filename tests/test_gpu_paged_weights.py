"""How exactly the paged attention weighs values: results that are small
beside their terms show what a weight was rounded to."""

import math

import numpy as np
import pytest
import torch

import _paged_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# significant bits of a stored value
BITS = {"fp16": 11, "bf16": 8, "fp8": 4}


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import paged

    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def _cancelling(fmt, w):
    """Values (..., n) of the tokens of sequences whose first token has weight
    w and the others 1, so that the weighted sum nearly vanishes: each value
    takes away as much of what is left as a row of the format holds.  INT4: one
    value in fp32, for rows whose elements are all the same hold that."""
    left, out = w.copy(), [np.ones_like(w)]
    for _ in range(1 if fmt == "fp8_int4" else -(-20 // BITS[fmt])):
        if fmt == "fp8_int4":
            c = left.astype(np.float32).astype(np.float64)
        else:
            m, e = np.frexp(left)
            c = np.ldexp(np.rint(np.ldexp(m, BITS[fmt])), e - BITS[fmt])
        out.append(-c)
        left = left - c
    return np.stack(out, -1)


@pytest.mark.parametrize("fmt,qd", [("bf16", "bf16"), ("fp8", "bf16"), ("fp8", "fp16"), ("fp8_int4", "bf16"),
                                    ("fp8_int4", "fp16")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,split", [(3, False), (3, True), (20, True)])
def test_weights_are_held_in_32_bits(paged, fmt, qd, D, G, split):
    """One weight w between 1/e and 1 beside weights of exactly 1.  What w may
    be off by, relative to it: log2(e) and its product with the score x, 2^-24
    each of the exponent, so x 2^-23; exp2, 2^-22; with a scale 2^-24.  Sums of
    N terms that are not zero (w enters as three), each addition off by
    2^-23 of the terms' magnitudes at most, and two more for the waves' join."""
    B, H, page = 8, 8, 16
    rng = np.random.default_rng(7)
    x = torch.from_numpy(rng.uniform(0.03, 1.0, (B, H))).to(DTYPES[qd])
    w = np.exp(-ref.f64(x))
    vals = _cancelling(fmt, w)
    n = vals.shape[-1]
    k, v = torch.zeros(B, H, n, D), torch.from_numpy(vals).float()[..., None].repeat(1, 1, 1, D)
    k[:, :, 0, 0] = -1.0
    if fmt == "fp8_int4":
        v[:, :, 0, ::2] = 0.0  # (a row that has a scale)
    layer = paged.PagedLayer(B, H, D, page, fmt)
    table = torch.arange(B, dtype=torch.int32).view(B, 1)
    layer.write(k.cuda(), v.cuda(), table.cuda(), 0)
    q = torch.zeros(B, H, G, D, dtype=DTYPES[qd])
    q[..., 0] = x[:, :, None]
    q = q.view(B, H * G, 1, D)
    # (a table of 1024 tokens is split, one of 16 not)
    wide = torch.cat([table, torch.full((B, 63), -1, dtype=torch.int32)], 1) if split else table
    got = layer.attend(q.cuda(), wide.cuda(), torch.full((B,), n, dtype=torch.int32, device="cuda"), scale=1.0)
    want, _, spread, _ = ref.attend(ref.f64(q)[:, :, 0], ref.page_values(layer), table.numpy(), [n] * B, page, B, 1.0)
    odd = np.abs(want)[..., 1::2]
    assert (odd <= 2.0 ** -19 * spread[..., 1::2]).all(), "the values do not cancel"
    terms = n + 2
    rel = 2.0 ** -23 * (1 + 2 + 0.5 + terms + 2)
    tol = (ref.UNIT[q.dtype] + 2.0 ** -20) * np.abs(want) + ref.TINY[q.dtype] + rel * spread
    err = np.abs(ref.f64(got)[:, :, 0] - want)
    assert (err <= tol).all(), f"error {(err / tol).max()} of the bound"
