"""Compiled calls of attention of several tokens, of attention over selected
pages and of the drafts' verification against the ones in Python: the same bits,
and nothing done for what they leave."""

import pytest
import torch

from test_gpu_paged_calls import _both, _i, _randn, paged  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

B, H, G, D, PAGE = 3, 2, 4, 64, 16


def _layer(paged, fmt="bf16", **kw):  # noqa: F811
    layer = paged.PagedLayer(24, H, D, PAGE, fmt, **kw)
    table = torch.randperm(24, generator=torch.Generator().manual_seed(2)).to("cuda", torch.int32).view(B, 8)
    dtype = paged._NEW.get(fmt, torch.float16)
    layer.write(_randn(3, B, H, 120, D, dtype=dtype), _randn(4, B, H, 120, D, dtype=dtype), table, 0)
    return layer, table, dtype


@pytest.mark.parametrize("fmt", ["fp16", "bf16", "fp8", "fp8_int4"])
def test_several_tokens(paged, monkeypatch, fmt):  # noqa: F811
    layer, table, dtype = _layer(paged, fmt)
    q, lens = _randn(5, B, H * G, 5, D, dtype=dtype), _i(120, 0, 37)
    strided = _randn(5, B, 5, H * G, D, dtype=dtype).transpose(1, 2)
    for kw in ({}, {"max_len": 64}, {"max_len": 10 ** 6}, {"lens_add": -2}, {"scale": 0.3}, {"scale": 1},
               {"return_lse": True}, {"n_new": _i(5, 0, 2)}, {"n_new": _i(5, 0, 2), "return_lse": True},
               {"n_new": _i(5, 0, 2), "out": torch.full_like(q, 7)}, {"out": torch.empty_like(q)},
               {"out": torch.empty_like(strided)}, {"shared": 32}, {"shared": PAGE * 8}):
        _both(monkeypatch, lambda: layer.attend_tokens(q, table, lens, **kw), True)
        _both(monkeypatch, lambda: layer.attend_tokens(strided, table, lens, **kw), True)
    for n in (0, 1, 70):
        many = _randn(6, B, H * G, n, D, dtype=dtype)
        _both(monkeypatch, lambda: layer.attend_tokens(many, table, lens), True)
    _both(monkeypatch, lambda: layer.attend_tokens(q[:0], table[:0], lens[:0], return_lse=True), True)
    _both(monkeypatch, lambda: layer.attend_tokens(q, table[:, ::2], lens), False)
    odd = _randn(5, B, H * G, 5, D + 8, dtype=dtype)[..., 1:D + 1]
    _both(monkeypatch, lambda: layer.attend_tokens(odd, table, lens), False)
    _both(monkeypatch, lambda: layer.attend_tokens(q, table, lens, n_new=_i(5, 1, 0, 1, 2, 1)[::2]), False)


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_selected_pages(paged, monkeypatch, fmt):  # noqa: F811
    layer, table, dtype = _layer(paged, fmt, bounds=True)
    q, lens = _randn(5, B, H * G, 1, D, dtype=dtype), _i(120, 0, 37)
    apart = _randn(5, B, H * G + 1, 1, D, dtype=dtype)[:, 1:]
    for kw in ({}, {"max_len": 64}, {"lens_add": -2}, {"scale": 0.3}, {"return_lse": True}, {"return_pages": True},
               {"return_lse": True, "return_pages": True}, {"out": torch.empty_like(q)}):
        for n_select in (1, 3, 100):
            _both(monkeypatch, lambda: layer.attend_sparse(q, table, lens, n_select, **kw), True)
        _both(monkeypatch, lambda: layer.attend_sparse(apart, table, lens, 3, **kw), False)
    _both(monkeypatch, lambda: layer.attend_sparse(q[:0], table[:0], lens[:0], 3, return_pages=True), True)
    _both(monkeypatch, lambda: layer.attend_sparse(q, table[:, ::2], lens, 3), False)


@pytest.mark.parametrize("fmt", ["fp16", "fp8_int4"])
def test_bounds(paged, monkeypatch, fmt):  # noqa: F811
    layer, table, _ = _layer(paged, fmt, bounds=True)
    want = layer.bounds.clone()
    wide = torch.cat([table, table], 1)

    def bound(*args):
        layer.bounds.zero_()
        layer.bound(*args)
        return [layer.bounds]

    for args, plain in (((table, 0, 120), True), ((table, 0, 0), True), ((table, _i(0, 3, 40), 9), True),
                        ((table, _i(0, 3, 40), 9, _i(9, 0, 2)), True), ((wide[:, :8], 5, 70), True),
                        ((table[:, ::2], 0, 60), False), ((table, 0, 9, _i(9, 1, 0, 1, 2, 1)[::2]), False)):
        got = _both(monkeypatch, lambda: [t.clone() for t in bound(*args)], plain)
        if args[2] == 120:
            assert torch.equal(got[0], want)
    for n in (-1, 2 ** 31):
        with pytest.raises(ValueError, match="n must be"):
            layer.bound(table, 0, n)


def test_refusals_are_worded_in_python(paged):  # noqa: F811
    layer, table, dtype = _layer(paged, bounds=True)
    q, lens = _randn(5, B, H * G, 5, D), _i(120, 0, 37)
    with pytest.raises(ValueError, match="whole pages"):
        layer.attend_tokens(q, table, lens, shared=8)
    with pytest.raises(ValueError, match="whole pages"):
        layer.attend_tokens(q, table, lens, shared=PAGE * 9)
    with pytest.raises(TypeError, match="queries"):
        layer.attend_tokens(q.half(), table, lens)
    with pytest.raises(ValueError, match="n_select"):
        layer.attend_sparse(q[:, :, :1], table, lens, 0)
    with pytest.raises(RuntimeError, match="scale"):
        layer.attend_sparse(q[:, :, :1], table, lens, 2, scale=-1.0)
    with pytest.raises(RuntimeError, match="requires grad"):
        layer.attend_tokens(q.requires_grad_(), table, lens)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 777, 40000])
def test_verification(monkeypatch, dtype, V):
    from foveated_kv_amd import drafts

    K = 4
    target = torch.softmax(_randn(1, B, K + 1, V, dtype=torch.float32), -1).to(dtype)
    draft = torch.softmax(_randn(2, B, K, V, dtype=torch.float32), -1).to(dtype)
    tokens = torch.randint(0, V, (B, K), generator=torch.Generator().manual_seed(3)).cuda()
    u = torch.rand((B, K + 1), generator=torch.Generator().manual_seed(4)).cuda()
    wide = torch.zeros((B, K + 2, V + 3), dtype=dtype, device="cuda")[:, 1:, 1:V + 1]
    wide.copy_(target)
    for t in (target, wide):
        for d in (draft, None):
            for toks in (tokens, tokens.int()):
                for n in (None, _i(4, 0, 2)):
                    _both(monkeypatch, lambda: drafts.verify_drafts(t, d, toks, u, n), True)
    _both(monkeypatch, lambda: drafts.verify_drafts(target, draft, tokens, u.t().contiguous().t(), None), False)
    _both(monkeypatch, lambda: drafts.verify_drafts(target[:0], None, tokens[:0], u[:0]), True)
    _both(monkeypatch, lambda: drafts.verify_drafts(target[:, :1], None, tokens[:, :0], u[:, :1].contiguous()), True)
