"""Selected pages of sequences with table entries outside the pool: the choice
fills up with these, the lower ones first, where the pages that are there are not
enough."""

import pytest
import torch

from test_gpu_paged import _bits_equal, _filled, _flush, _randn, _table
from test_gpu_paged_sparse import _check, _i32, _with_bounds, paged  # noqa: F401

pytestmark = pytest.mark.gpu


def _dirty():
    """Memory that calls to come will have as workspace: ids of page 0."""
    torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("pages,holes", [(10, [2, 5]), (10, [0, 1, 7]), (9, [3, 4, 5, 6]), (40, [0, 11, 38]), (64, [1, 2, 62]),
                                         (65, list(range(1, 60, 2))), (200, [5, 100, 101, 198]), (1500, list(range(3, 1490, 90)))])
def test_more_pages_wanted_than_there_are(paged, fmt, pages, holes):  # noqa: F811
    _flush("holes", fmt, pages, len(holes))
    page, H, G, D = 16, 2, 3, 64
    layer = _with_bounds(paged, _filled(paged, fmt, pages + 3, H, D, page, 90))
    table = _table(91, pages + 3, [pages])
    layer.bound(table.cuda(), 0, pages * page)
    for j, i in enumerate(holes):
        table[0, i] = [-1, 2 ** 30, pages + 3][j % 3]
    q = _randn(92, 1, H * G, 1, D).bfloat16().cuda()
    there = pages - 1 - len(holes)
    for n_select in sorted({2, there, there + 1, there + 2, there + 3, pages - 1, pages, pages + 2}):
        if n_select > 0:
            _dirty()
            _check(layer, q, table, [pages * page - 5], n_select)


@pytest.mark.parametrize("pages,holes", [(20, [0, 4]), (65, [7, 8, 30]), (300, list(range(0, 290, 7)))])
def test_equal_scores_and_holes(paged, pages, holes):  # noqa: F811
    page, D = 16, 64
    layer = _with_bounds(paged, paged.PagedLayer(pages, 1, D, page, "bf16"))
    layer.k.fill_(0.5)
    layer.v.copy_(_randn(93, pages, 1, page, D))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(94)).int().view(1, pages)
    layer.bound(table.cuda(), 0, pages * page)
    table[0, holes] = -1
    q = torch.ones(1, 2, 1, D, dtype=torch.bfloat16, device="cuda")
    there = pages - 1 - len(holes)
    first = None
    for n_select in (3, there + 1, there + 2, there + len(holes), pages - 1, pages):
        _dirty()
        out = _check(layer, q, table, [pages * page], n_select)
        if n_select > there:  # (pages that are not there add nothing)
            first = out if first is None else first
            assert bool(torch.allclose(out.float(), first.float(), atol=2.0 ** -7))
    full = layer.attend(q, table.cuda(), _i32([pages * page]))
    assert bool(torch.allclose(first.float(), full.float(), atol=2.0 ** -7))
    _dirty()
    _bits_equal(_check(layer, q, table, [pages * page], pages - 1), _check(layer, q, table, [pages * page], pages - 1), "again")
