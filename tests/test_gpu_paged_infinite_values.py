"""Infinite values among the tokens that a query attends to: infinity of their sign
in that dim, wherever in the tiles and parts of the tokens they lie."""

import math

import pytest
import torch

from test_gpu_paged import DTYPES, _bits_equal, _filled, _flush, _randn, _table
from test_gpu_paged_tokens import KINDS, _i32, paged  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,qd", [kind for kind in KINDS if kind[0] != "fp8"])  # (E4M3 values are finite or NaN)
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("D,G,L,shared", [(128, 3, 6, 0), (64, 7, 6, 0), (128, 3, 6, 16), (128, 4, 90, 0)])
def test_infinite_values_keep_their_sign(paged, fmt, qd, bad, D, G, L, shared):  # noqa: F811
    _flush("infinite", fmt, qd, bad, D, G, L, shared)
    page, H = 16, 1
    lens = [max(40, L + 5), 133, L + shared, 1500]
    counts = [-(-n // page) for n in lens]
    layer = _filled(paged, fmt, sum(counts), H, D, page, 60)
    table = _table(61, sum(counts), counts)
    if shared:
        table[:, 0] = table[0, 0]
    on, n = table.cuda(), _i32(lens)
    q = _randn(62, len(lens), H * G, L, D).to(DTYPES[qd]).cuda()
    want = layer.attend_tokens(q, on, n, shared=shared)
    for hit in (0, 3, L - 1):  # the new token with the bad value
        for b, length in enumerate(lens):
            p = length - L + hit
            at = (int(table[b, p // page]), 0, p % page)
            t = layer.v_scale if fmt == "fp8_int4" else layer.v
            dim = 1 if fmt == "fp8_int4" else 5
            kept = t[at].clone()
            t[at][dim] = bad
            for kw in ({}, {"max_len": max(lens)}):
                got = layer.attend_tokens(q, on, n, shared=shared, **kw)[b].float()
                late = got[:, hit:] if fmt == "fp8_int4" else got[:, hit:, 5]
                assert bool((late == bad).all()), f"token {hit} of {length}: {late.flatten()[:4].tolist()}"
                if not kw:
                    _bits_equal(got[:, :hit], want[b, :, :hit].float(), "before")
                    if fmt != "fp8_int4":
                        _bits_equal(got[..., :5], want[b, ..., :5].float(), "other dims")
            t[at] = kept
    _bits_equal(layer.attend_tokens(q, on, n, shared=shared), want, "restored")
