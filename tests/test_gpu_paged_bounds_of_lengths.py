"""Attention by the C entry points with a bound of the lengths beyond what any
table holds: what a bound that the table's width gives computes, to the bounds of
the 64-bit restatement's tests."""

import ctypes

import pytest
import torch

from test_gpu_paged import _bits_equal, _filled, _flush, _randn, _table
from test_gpu_paged_tokens import _i32, paged  # noqa: F401

pytestmark = pytest.mark.gpu


def _rows(t):
    from foveated_kv_amd import _lib

    return _lib.RowsC(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


@pytest.mark.parametrize("L,lens", [(5, [1900]), (5, [700, 0, 3, 900, 64, 65, 1500]), (300, [1000, 301])])
@pytest.mark.parametrize("max_len", [2 ** 31 - 4096, 2 ** 36, 2 ** 40, 2 ** 63 - 1])
def test_several_tokens(paged, L, lens, max_len):  # noqa: F811
    from foveated_kv_amd import _lib

    _flush("bound", L, lens, max_len)
    B, H, G, D, page = len(lens), 2, 4, 128, 64
    counts = [max(1, -(-n // page)) for n in lens]
    layer = _filled(paged, "bf16", sum(counts), H, D, page, 10)
    table = _table(11, sum(counts), counts).cuda()
    q = _randn(12, B, H * G, L, D).bfloat16().cuda()
    want, want_lse = layer.attend_tokens(q, table, _i32(lens), max_len=2 ** 40, return_lse=True)
    lib = _lib.load()

    def call(bound):
        out, lse, n = torch.empty_like(q), torch.empty(B, H * G, L, device="cuda"), _i32(lens)
        size = lib.fkv_paged_attn_rows_workspace(layer._c, H * G, B, L, 0, bound)
        ws = torch.full((max(size, 1),), 85, dtype=torch.uint8, device="cuda")
        rc = lib.fkv_paged_attn_rows(layer._c, ctypes.byref(_rows(q)), 1, H * G, B, L, table.data_ptr(), table.shape[1],
                                     table.stride(0), n.data_ptr(), 0, None, 0, bound, D ** -0.5, ctypes.byref(_rows(out)),
                                     lse.data_ptr(), ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.fkv_last_error()
        torch.cuda.synchronize()
        return out, lse

    out, lse = call(max_len)
    for a, b in zip((out, lse), call(2 ** 31 - 4096)):
        _bits_equal(a, b, "the longest bound")
    # (parts of other lengths: sums in another order, and a bf16 weight and result each)
    assert bool(((out.float() - want.float()).abs() <= 2.0 ** -6 * (1 + want.float().abs())).all())
    real = ~torch.isinf(want_lse)
    assert torch.equal(real, ~torch.isinf(lse)) and bool(((lse - want_lse).abs()[real] <= 1e-4).all())


@pytest.mark.parametrize("max_len", [2 ** 36, 2 ** 63 - 1])
def test_one_token(paged, max_len):  # noqa: F811
    from foveated_kv_amd import _lib

    lens, H, G, D, page = [1900, 700], 2, 4, 128, 64
    layer = _filled(paged, "fp8", 41, H, D, page, 20)
    table = _table(21, 41, [30, 11]).cuda()
    q = _randn(22, 2, H * G, 1, D).half().cuda()
    want = layer.attend(q, table, _i32(lens))
    lib = _lib.load()
    out, n = torch.empty_like(q), _i32(lens)
    size = lib.fkv_paged_attn_workspace(layer._c, H * G, 2, max_len)
    ws = torch.full((size,), 85, dtype=torch.uint8, device="cuda")
    rc = lib.fkv_paged_attn(layer._c, ctypes.byref(_rows(q)), 0, H * G, 2, table.data_ptr(), table.shape[1], table.stride(0),
                            n.data_ptr(), 0, max_len, D ** -0.5, out.data_ptr(), None, ws.data_ptr(), size,
                            torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.fkv_last_error()
    # (two fp32 sums of other parts, each rounded to fp16)
    assert bool(((out.float() - want.float()).abs() <= 2.0 ** -9 * (1 + want.float().abs())).all())
