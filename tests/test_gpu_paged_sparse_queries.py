"""Queries of one KV head over selected pages, whatever the strides between
sequences and of dimensions of one element."""

import pytest
import torch

from test_gpu_paged import _bits_equal, _filled, _flush, _randn, _table
from test_gpu_paged_sparse import _check, _i32, _with_bounds, paged  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq", [1, 3, 20])
def test_strides_of_one_kv_head(paged, Hq):  # noqa: F811
    _flush("one head", Hq)
    page, D, B = 16, 64, 5
    lens = [310, 77, 0, 16, 200]
    counts = [-(-n // page) for n in lens]
    layer = _with_bounds(paged, _filled(paged, "bf16", sum(counts), 1, D, page, 80))
    table = _table(81, sum(counts), counts)
    layer.bound(table.cuda(), 0, max(lens), n_new=_i32(lens))
    q = _randn(82, B, Hq, 1, D).bfloat16().cuda()
    want = _check(layer, q, table, lens, 6)
    views = [torch.zeros(Hq, B, 1, D, dtype=q.dtype, device="cuda").transpose(0, 1),
             torch.zeros(B, Hq + 2, 1, D, dtype=q.dtype, device="cuda")[:, 1:Hq + 1],
             torch.zeros(B, Hq, 7, D, dtype=q.dtype, device="cuda")[:, :, 3:4],
             torch.zeros(B, Hq, 1, D + 8, dtype=q.dtype, device="cuda")[..., :D],
             torch.zeros(B, Hq, 1, D + 3, dtype=q.dtype, device="cuda")[..., 1:D + 1]]
    if Hq == 1:
        views.append(torch.zeros(B * D, dtype=q.dtype, device="cuda").as_strided((B, 1, 1, D), (D, 3, 5, 1)))
    for x in views:
        x.copy_(q)
        _bits_equal(layer.attend_sparse(x, table.cuda(), _i32(lens), 6), want, x.stride())
    x = q.clone()
    assert layer.attend_sparse(x, table.cuda(), _i32(lens), 6, out=x) is x
    _bits_equal(x, want, "in place")
    # the compiled call takes what needs no copy
    from foveated_kv_amd import _lib

    for x in views[:3]:
        done = _lib.calls().attend_sparse(layer._key, layer.bounds, x, table.cuda(), _i32(lens), 6, None, 0, None, None, False,
                                          False)
        assert done is not NotImplemented
        _bits_equal(done, want, x.stride())
