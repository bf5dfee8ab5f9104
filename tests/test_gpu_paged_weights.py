"""How exactly the paged attention weighs values: results that are small
beside their terms show what a weight was rounded to."""

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


@pytest.mark.parametrize("fmt,qd", [("fp16", "fp16"), ("bf16", "bf16"), ("fp8", "bf16"), ("fp8", "fp16"),
                                    ("fp8_int4", "bf16"), ("fp8_int4", "fp16")])
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


@pytest.mark.parametrize("fmt,qd", [("fp16", "fp16"), ("bf16", "bf16"), ("fp8", "fp16"), ("fp8_int4", "bf16")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G", [(40, 4), (512, 4), (1500, 4), (1500, 20)])
def test_a_token_above_the_others_whose_value_is_zero(paged, fmt, qd, D, n, G):
    """A sink: it has nearly all of the weight and adds nothing, so that the
    result is the others', whose weights are e^-10 and less of its own."""
    above = [10.0, 14.0, 16.0, 18.0, 20.0, 24.0]  # nats, of each sequence's first token
    B, H, page = len(above), 2, 16
    P = -(-n // page)
    g = torch.Generator().manual_seed(n + D + G)
    k, v = torch.randn(B, H, n, D, generator=g), torch.randn(B, H, n, D, generator=g) * 2.0 ** 12
    q = torch.randn(B, H * G, 1, D, generator=g)
    k[..., 0] = 0.0
    q[..., 0] = 4.0
    k[:, :, 0] = 0.0
    k[:, :, 0, 0] = torch.tensor(above)[:, None] * D ** 0.5 / 4.0
    v[:, :, 0] = 0.0
    layer = paged.PagedLayer(B * P, H, D, page, fmt)
    table = torch.arange(B * P, dtype=torch.int32).view(B, P)
    layer.write(k.cuda(), v.cuda(), table.cuda(), 0)
    q = q.to(DTYPES[qd])
    got, lse = layer.attend(q.cuda(), table.cuda(), torch.full((B,), n, dtype=torch.int32, device="cuda"),
                            return_lse=True)
    want, wlse, spread, ds = ref.attend(ref.f64(q)[:, :, 0], ref.page_values(layer), table.numpy(), [n] * B, page,
                                        B * P, D ** -0.5)
    tol = ref.attend_bound(want, spread, ds, [n] * B, q.dtype)
    err = np.abs(ref.f64(got)[:, :, 0] - want)
    # (24 nats leave results that end in the result type's smallest numbers)
    assert np.abs(want[:3]).max(-1).min() > 1e3 * ref.TINY[q.dtype], "too small to see"
    assert (err <= tol).all(), f"error {(err / tol).max()} of the bound"
    assert (np.abs(ref.f64(lse) - wlse) <= 2 * ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(wlse)).all()


@pytest.mark.parametrize("fmt", ["fp16", "bf16"])
@pytest.mark.parametrize("scores", [2.0 ** 27 + 2.0 ** 14, 2.0 ** 26 + 2.0 ** 14, 2.0 ** 24 + 2.0 ** 14])
def test_scores_whose_steps_are_as_large_as_the_slack(paged, fmt, scores):
    """Scores (in powers of two) with a step of 16 or 8 beside a running
    maximum that lets them pass it by 15: the later token, 16 above the earlier
    one, has a weight of 2^16 of it, and the result is its value but for that."""
    D, page, n = 64, 16, 256
    half = scores - 2.0 ** 14
    layer = paged.PagedLayer(n // page, 1, D, page, fmt)
    k, v = torch.zeros(1, 1, n, D), torch.zeros(1, 1, n, D)
    k[..., 0], k[..., 1] = half / 2.0 ** 13, 2.0 ** 7
    k[:, :, 1:] *= -1.0  # (far below: no weight)
    k[:, :, 128] = k[:, :, 0]
    k[:, :, 128, 2] = 4.0
    v[:, :, 0], v[:, :, 128] = 3.0, 5.0
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").view(1, -1)
    layer.write(k.cuda(), v.cuda(), table, 0)
    q = torch.zeros(1, 2, 1, D, dtype=DTYPES[fmt])
    q[..., 0], q[..., 1], q[..., 2] = 2.0 ** 13, 2.0 ** 7, 4.0
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    # (the scale times log2 e is 1 or next to it: scores off by 2^-23 of themselves, 16 at most)
    for wide in (table, torch.nn.functional.pad(table, (0, 64), value=-1)):  # (a table of 1280 tokens is split)
        out = layer.attend(q.cuda(), wide, lens, scale=float(np.log(2.0)))
        assert bool(((out.float() - 5.0).abs() <= 5.0 * ref.UNIT[q.dtype] + 2.0 * 2.0 ** -15).all()), out.unique()
