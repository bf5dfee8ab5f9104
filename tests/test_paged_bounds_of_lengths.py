"""Bounds of the lengths beyond what a table can hold: a launch is planned as for
the longest sequences that there can be."""

import ctypes

import pytest

from foveated_kv_amd import _lib

MOST = 2 ** 31 - 4096
R = ctypes.byref


def _pages(H, D=128, fmt=1):
    exps = 4096 if fmt > 1 else None
    return _lib.PagesC(4096, 4096, exps, exps, 1000, 64, H, D, fmt)


@pytest.mark.parametrize("H,Hq,B,L,shared", [(8, 32, 1, 5, 0), (8, 32, 32, 5, 0), (8, 32, 4, 2048, 0), (8, 32, 64, 1, 16384),
                                             (1, 1, 1, 1, 0), (2, 14, 7, 3, 1024)])
@pytest.mark.parametrize("D,fmt", [(128, 1), (64, 0), (128, 3)])
def test_workspaces_of_lengths_beyond_the_most(H, Hq, B, L, shared, D, fmt):
    lib, pg = _lib.load(), _pages(H, D, fmt)
    for size in (lambda n: lib.fkv_paged_attn_rows_workspace(R(pg), Hq, B, L, shared, n),
                 lambda n: lib.fkv_paged_attn_workspace(R(pg), Hq, B, n),
                 lambda n: lib.fkv_paged_attn_sparse_workspace(R(pg), Hq, B, 100, 7, n)):
        want = size(MOST)
        assert want >= 0
        for n in (MOST + 1, 2 ** 31, 2 ** 36, 2 ** 40, 2 ** 62, 2 ** 63 - 1):
            assert size(n) == want, n


@pytest.mark.parametrize("n_table", [0, 1, 7, 500])
def test_workspaces_of_more_pages_than_there_are(n_table):
    """As many pages as a table holds are selected at most, and no more is kept for
    them."""
    lib, pg = _lib.load(), _pages(8)

    def size(n_select):
        return lib.fkv_paged_attn_sparse_workspace(R(pg), 32, 64, n_table, n_select, MOST)

    for n in (n_table + 1, 1000, 100000):
        assert size(n) == size(max(n_table, 1)) > 0
