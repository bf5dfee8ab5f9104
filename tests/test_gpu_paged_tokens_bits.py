"""How many bits of a weight reach the results of attention of several tokens: as
many for tokens far below the row's largest as for others, and as many behind a
shared beginning as elsewhere."""

import numpy as np
import pytest
import torch

import _paged_ref as ref
from test_gpu_paged import DTYPES, _filled, _flush, _randn, _table
from test_gpu_paged_tokens import KINDS, _i32, _values, paged  # noqa: F401

pytestmark = pytest.mark.gpu

# a weight as the sum of two 16-bit numbers: bf16 pages the upper half, which leaves less than
# 2^-7, and that rounded to 8 bits, 2^-16; fp16 pages 11 bits cut off, which leaves less than
# 2^-10, and that rounded to 11, 2^-21, or 2^-46 of the row's largest weight; quantised ones
# two bf16 numbers, both rounded, 2^-9 and 2^-18
PART = {"bf16": 2.0 ** -16, "fp16": 2.0 ** -21, "fp8": 2.0 ** -18, "fp8_int4": 2.0 ** -18}


def _tight(out, spread, ds, n, fmt, dtype, mag):
    """A result's own rounding; per weight the score's error (twice, once in the
    sum), exp2's and the sum's (2^-21) and its two numbers'; fp32 sums of four
    products of 16 tokens for every 32, each rounded twice at most, then waves and
    workgroups."""
    rel = 2 * ds + PART[fmt] + 2.0 ** -21 + (n / 4 + 64) * 2.0 ** -24
    small = n * 2.0 ** -46 * mag if fmt == "fp16" else 0.0
    return ref.UNIT[dtype] * np.abs(out) + ref.TINY[dtype] + rel * spread + small


@pytest.mark.parametrize("fmt,qd", KINDS)
@pytest.mark.parametrize("D,G,L,shared", [(128, 4, 3, 0), (64, 7, 3, 0), (128, 4, 100, 0), (64, 4, 70, 0), (128, 4, 1, 256),
                                          (64, 8, 2, 64)])
def test_bits_of_weights(paged, fmt, qd, D, G, L, shared):  # noqa: F811
    """Keys of few values, so that scores are exact: 64-bit results to within the
    weights' own errors."""
    _flush("bits", fmt, qd, D, G, L, shared)
    page, H, lens = 16, 2, [700, 333, 128, 97]
    lens = [n + shared for n in lens] if shared else [max(n, L) for n in lens]
    counts = [-(-n // page) for n in lens]
    layer = _filled(paged, fmt, sum(counts), H, D, page, 90)
    gen = torch.Generator().manual_seed(91)
    levels = torch.randint(-6, 7, (sum(counts), H, page), generator=gen).float()
    k = torch.zeros(sum(counts), H, page, D)
    k[..., 0] = levels * 0.5  # (in E4M3 exact whatever power of two goes with them)
    v = _randn(92, sum(counts), H, page, D)
    ids = torch.arange(sum(counts), dtype=torch.int32, device="cuda").view(-1, 1)
    layer.write(k.cuda(), v.cuda(), ids, 0)
    table = _table(93, sum(counts), counts)
    if shared:
        table[:, :shared // page] = table[0, :shared // page]
    q = torch.zeros(len(lens), H * G, L, D)
    q[..., 0] = torch.randint(1, 5, (len(lens), H * G, L), generator=gen).float()
    q = q.to(DTYPES[qd]).cuda()
    out = ref.f64(layer.attend_tokens(q, table.cuda(), _i32(lens), scale=0.5, shared=shared))
    values, q64, t = _values(layer), ref.f64(q), table.numpy()
    mag = float(np.abs(values[1]).max())
    for l in range(0, L, max(1, L // 9)):
        limit = [n - L + l + 1 for n in lens]
        want, _, spread, _ = ref.attend(q64[:, :, l], values, t, limit, page, layer.n_pages, 0.5)
        # scores up to 6: the factor's rounding, the product's with the maximum taken off
        tol = _tight(want, spread, 4 * 2.0 ** -24 * 6, max(lens), fmt, DTYPES[qd], mag)
        err = np.abs(out[:, :, l] - want)
        assert (err <= tol).all(), f"token {l}: {(err / tol).max()} of the bound"


@pytest.mark.parametrize("fmt,qd", KINDS)
@pytest.mark.parametrize("nats", [8, 14, 17, 20, 24])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_bits_below_a_dominating_token(paged, fmt, qd, nats, where):  # noqa: F811
    """One token far above the others, of value zero: the result is made of the
    others' weights, and as exact as it is without that token."""
    _flush("below", fmt, qd, nats, where)
    page, D, n, L = 16, 128, 200, 3
    layer = paged.PagedLayer(13, 1, D, page, fmt)
    k = torch.zeros(1, 1, n, D)
    at = {"first": 0, "middle": 77, "last": n - L}[where]
    k[0, 0, at, 0] = 16.0
    v = _randn(71, 1, 1, n, D)
    v = v * (20000.0 / float(v.abs().max()))
    v[0, 0, at] = 0.0
    table = torch.arange(13, dtype=torch.int32).view(1, 13)
    layer.write(k.cuda(), v.cuda(), table.cuda(), 0)
    q = torch.zeros(1, 4, L, D)
    q[..., 0] = 1.0
    q = q.to(DTYPES[qd]).cuda()
    scale = nats / 16
    values, q64 = _values(layer), ref.f64(q)
    mag = float(np.abs(values[1]).max())
    for B, shared in ((1, 0), (2, 96)):
        out = ref.f64(layer.attend_tokens(q.expand(B, -1, -1, -1), table.expand(B, -1).cuda(), _i32([n] * B), scale=scale,
                                          shared=shared))
        for l in range(L):
            want, _, spread, _ = ref.attend(q64[:, :, l], values, table.numpy(), [n - L + l + 1], page, 13, scale)
            tol = _tight(want, spread, 4 * 2.0 ** -24 * nats, n, fmt, DTYPES[qd], mag)
            err = np.abs(out[:, :, l] - want)
            assert (err <= tol).all(), f"token {l}: {(err / tol).max()} of the bound"


@pytest.mark.parametrize("fmt,qd", KINDS)
def test_one_token_behind_a_shared_beginning(paged, fmt, qd):  # noqa: F811
    """The cache's one-token call with and without a beginning held in common: two
    results that are each within a rounding of the exact one, or a bit more."""
    _flush("shared bits", fmt, qd)
    dt, B, H, G, D, page = DTYPES[qd], 5, 2, 4, 128, 16
    k, v = _randn(10, 1, H, 512, D).to(dt).cuda(), _randn(11, 1, H, 512, D).to(dt).cuda()
    own = [(_randn(20 + b, 1, H, 40 + 7 * b, D).to(dt).cuda(), _randn(30 + b, 1, H, 40 + 7 * b, D).to(dt).cuda()) for b in range(B)]
    q = _randn(12, B, H * G, 1, D).to(dt).cuda()
    outs = []
    for share in (False, True):
        cache = paged.PagedKVCache(1, H, D, 300, max_seqs=B, max_tokens=640, page_size=page, fmt=fmt)
        for b in range(B):
            one = slice(b, b + 1)
            if share and b:
                cache.share(0, 512, one)
            else:
                cache.extend(512, one)
                cache.write(0, k, v, seqs=one)
        for b in range(B):
            one = slice(b, b + 1)
            cache.extend(own[b][0].shape[2], one)
            cache.write(0, *own[b], seqs=one)
        assert cache.pages.common_tokens() == (512 if share else 0)
        outs.append(cache.attend(0, q).float())
    # a rounding each, and the weights' errors (relative to sums of magnitudes: some 1 here)
    tol = 2 * ref.UNIT[dt] * outs[0].abs() + 2.0 ** -15
    assert bool(((outs[0] - outs[1]).abs() <= tol).all())
    # few are rounded otherwise at all: those whose exact value lies near a border
    assert float((outs[0] != outs[1]).float().mean()) < 0.05
