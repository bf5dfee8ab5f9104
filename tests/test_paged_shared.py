"""The paged cache's shared beginnings, taken-back tokens and further entry
points without a GPU: bookkeeping and every refusal of the C entry points."""

import ctypes
import math
import random

import pytest
import torch

from foveated_kv_amd import PagedKVCache, PageTable, _lib
from test_paged import BAD_PAGES, R, _refused, c  # noqa: F401


def _check(t):
    holders = [0] * t.n_pages
    for b in range(t.max_seqs):
        for p in t.pages(b):
            holders[p] += 1
        row, n = t.table[b].tolist(), len(t.pages(b))
        assert row[:n] == t.pages(b) and all(x == -1 for x in row[n:]) and len(set(t.pages(b))) == n
        assert t.lens[b] == t.lengths()[b] <= n * t.page_size
        assert t.start[b] == t.starts()[b] and t.new[b] == t.lens[b] - t.start[b] >= 0
    assert holders == t._holders and sorted(t._free) == [p for p in range(t.n_pages) if holders[p] == 0]
    for first in range(t.max_seqs):
        for stop in range(first, t.max_seqs + 1):
            rows, n = [t.pages(b) for b in range(first, stop)], 0
            if len(rows) > 1:
                while all(len(r) > n and r[n] == rows[0][n] for r in rows):
                    n += 1
            assert t.common_tokens(slice(first, stop)) == n * t.page_size


def test_share_and_free():
    t = PageTable(20, 16, 4, 160, device="cpu")
    t.extend(50, slice(0, 1))
    t.share(0, 32, slice(1, 3))
    _check(t)
    assert t.lengths() == [50, 32, 32, 0] and t.starts() == [0, 32, 32, 0] and t.free_pages == 16
    assert t.common_tokens(slice(0, 3)) == 32 and t.common_tokens() == 0
    t.extend([3, 1, 17, 0])
    _check(t)
    assert t.pages(1)[:2] == t.pages(0)[:2] and t.pages(1)[2] != t.pages(0)[2]
    t.share(2, 48, slice(3, 4))
    _check(t)
    assert t.common_tokens(slice(2, 4)) == 48 and t.common_tokens() == 32
    t.free(0)
    _check(t)
    assert t.common_tokens(slice(1, 3)) == 32 and t.pages(1)[:2] == t.pages(2)[:2]
    t.free(2)
    t.free(1)
    _check(t)
    assert t.free_pages == 20 - 3 and t.lengths()[3] == 48
    t.free(3)
    _check(t)
    assert t.free_pages == 20


def test_rollback():
    t = PageTable(20, 16, 3, 160, device="cpu")
    t.extend([40, 20, 0])
    t.extend([5, 5, 0])
    t.rollback([3, 5, 0])
    _check(t)
    assert t.lengths() == [42, 20, 0] and t.starts() == [40, 20, 0] and t.new.tolist() == [2, 0, 0]
    t.rollback(0)
    t.rollback([10, 20, 0])  # past the last extend, and to nothing
    _check(t)
    assert t.lengths() == [32, 0, 0] and t.starts() == [32, 0, 0] and len(t.pages(0)) == 3
    t.extend([20, 1, 1])
    _check(t)
    assert t.lengths() == [52, 1, 1] and len(t.pages(0)) == 4
    t.free(2)
    t.share(0, 48, slice(2, 3))
    before = t.lengths()
    for bad in (lambda: t.rollback([5, 0, 0]), lambda: t.rollback([0, 0, 1]), lambda: t.rollback([0, 2, 0]),
                lambda: t.rollback(-1), lambda: t.rollback([0, 0])):
        with pytest.raises(ValueError):
            bad()
        assert t.lengths() == before
        _check(t)
    t.rollback([4, 0, 0])  # (48 tokens are left, the shared ones)
    _check(t)
    t.free(2)
    t.rollback([40, 0, 0])
    _check(t)


@pytest.mark.parametrize("kw", [dict(src=4, tokens=16), dict(src=-1, tokens=16), dict(src=0, tokens=17), dict(src=0, tokens=-16),
                                dict(src=0, tokens=64), dict(src=1, tokens=16), dict(src=0, tokens=16, seqs=slice(0, 2)),
                                dict(src=0, tokens=16, seqs=slice(0, 4, 2))])
def test_share_refusals(kw):
    t = PageTable(20, 16, 4, 160, device="cpu")
    t.extend(50, slice(0, 1))
    with pytest.raises(ValueError):
        t.share(kw["src"], kw["tokens"], kw.get("seqs", slice(2, 3)))
    _check(t)
    t.share(0, 0, slice(2, 3))
    t.share(0, 32, slice(2, 2))
    assert t.lengths() == [50, 0, 0, 0]
    with pytest.raises(TypeError):
        t.share(0, 16.0, slice(2, 3))


def test_any_order():
    """Random calls against the definition of what is held."""
    rng = random.Random(5)
    t = PageTable(40, 16, 5, 200, device="cpu")
    for _ in range(400):
        what, b = rng.random(), rng.randrange(5)
        try:
            if what < 0.4:
                t.extend([rng.randrange(30) if rng.random() < 0.5 else 0 for _ in range(5)])
            elif what < 0.6:
                t.share(b, rng.randrange(6) * 16, slice(rng.randrange(5), rng.randrange(6)))
            elif what < 0.8:
                t.rollback([rng.randrange(10) for _ in range(5)])
            elif what < 0.9:
                t.reserve(rng.randrange(200), slice(b, b + 1))
            else:
                t.free(b)
        except (ValueError, MemoryError):
            pass
        _check(t)


def test_cache_arguments():
    with pytest.raises(ValueError, match="sparse_pages"):
        PagedKVCache(1, 1, 128, 4, sparse_pages=-1, device="cpu")
    with pytest.raises(TypeError):
        PagedKVCache(1, 1, 128, 4, sparse_pages=1.5, device="cpu")


def test_shared_beginnings_of_prompts():
    from foveated_kv_amd.generate import _common_tokens

    assert _common_tokens([[1] * 40, [1] * 40], 16) == 32
    assert _common_tokens([[1] * 32, [1] * 40], 16) == 16  # (each prompt keeps a token of its own)
    assert _common_tokens([[1] * 33, [1] * 20 + [2] * 20], 16) == 16
    assert _common_tokens([[1], [1]], 16) == 0 and _common_tokens([[2] * 40, [1] * 40], 16) == 0


def test_drafting_arguments():
    from foveated_kv_amd import generate

    class Tok:
        def encode(self, text):
            return [1, 2]

    class Cache:
        rope, pages = 1, PageTable(4, 16, 2, 32, device="cpu")

    class Model:
        def parameters(self):
            return iter([torch.zeros(1)])

    a, b = Cache(), Cache()
    b.rope = None
    for kw in (dict(draft_model=Model()), dict(draft_cache=a), dict(draft_model=Model(), draft_cache=a),
               dict(draft_model=Model(), draft_cache=b), dict(draft_model=Model(), draft_cache=Cache(), n_draft=0),
               dict(draft_model=Model(), draft_cache=Cache(), n_draft=64)):
        with pytest.raises(ValueError, match="draft"):
            generate.generate_paged(Model(), Tok(), ["x"], a, **kw)


# ---------------------------------------------------------------------------
# C entry points
# ---------------------------------------------------------------------------

def _rows_call(c, pages=None, **kw):
    a = dict(format=2, q={}, q_dtype=0, Hq=4, B=1, L=3, table=c.at, n_table=64, stride=2 ** 27, lens=c.at, n_new=None, shared=0,
             max_len=65536, scale=1.0, out={"data": c.at + 4096}, ws=c.at, ws_bytes=1 << 50)
    a.update(kw)
    pages = c.pages(format=a["format"]) if pages is None else pages
    q, out = (None if a[n] is None else R(c.rows(**{"stride_b": 4 * 64 * 8, "stride_h": 64 * 8, **a[n]})) for n in ("q", "out"))
    return c.lib.fkv_paged_attn_rows(None if pages == 0 else R(pages), q, a["q_dtype"], a["Hq"], a["B"], a["L"], a["table"],
                                     a["n_table"], a["stride"], a["lens"], 0, a["n_new"], a["shared"], a["max_len"], a["scale"],
                                     out, None, a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("word,kw", [
    ("sequences", {"B": 4097}), ("sequences", {"B": -1}), ("multiple", {"Hq": 3}), ("multiple", {"Hq": 0}), ("2^28", {"L": -1}),
    ("2^28", {"L": 2 ** 27}), ("max_len", {"max_len": -1}), ("whole pages", {"shared": -16}), ("whole pages", {"shared": 24}),
    ("more shared", {"shared": 65 * 16}), ("table shape", {"n_table": -1}), ("2^31 tokens", {"n_table": 2 ** 27}),
    ("fp16 or bf16", {"q_dtype": 2}), ("16-bit pages' type", {"format": 0, "q_dtype": 1}),
    ("16-bit pages' type", {"format": 1, "q_dtype": 0}), ("finite", {"scale": math.nan}), ("NULL", {"q": None}),
    ("NULL", {"out": None}), ("NULL", {"lens": None}), ("aligned", {"q": {"data": 0x1008}}), ("aligned", {"out": {"data": 0x1008}}),
    ("multiples", {"q": {"stride_h": 60}}), ("multiples", {"out": {"stride_l": 4}}), ("workspace", {"ws": None}),
    ("workspace", {"ws_bytes": 16}), ("aligned", {"ws": 0x1004}), ("NULL table", {"table": None}),
    ("rows of out share", {"out": {"stride_l": 32}}), ("share memory", {"out": {"data": None}})])
def test_rows_refusals(c, word, kw):  # noqa: F811
    if word == "share memory":
        kw = {"out": {"data": c.at + 128}}
    _refused(_rows_call(c, **kw), c.lib, word)


def _sparse_call(c, pages=None, **kw):
    a = dict(format=2, bounds=c.at, q={}, q_dtype=0, Hq=4, B=2, table=c.at, n_table=64, stride=2 ** 27, lens=c.at, max_len=1024,
             k=4, scale=1.0, out=c.at + 4096, ws=c.at, ws_bytes=1 << 50)
    a.update(kw)
    pages = c.pages(format=a["format"]) if pages is None else pages
    return c.lib.fkv_paged_attn_sparse(None if pages == 0 else R(pages), a["bounds"],
                                       None if a["q"] is None else R(c.rows(**{"stride_b": 256, **a["q"]})), a["q_dtype"], a["Hq"],
                                       a["B"], a["table"], a["n_table"], a["stride"], a["lens"], 0, a["max_len"], a["k"], a["scale"],
                                       a["out"], None, None, a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("word,kw", [
    ("4096 sequences", {"B": 2049}), ("4096 sequences", {"B": -1}), ("multiple", {"Hq": 3}), ("max_len", {"max_len": -1}),
    ("one page", {"k": 0}), ("one page", {"k": 2 ** 27}), ("table shape", {"n_table": 70, "stride": 69}),
    ("2^31 tokens", {"n_table": 2 ** 27}), ("2^31 tiles", {"B": 2048, "k": 2 ** 24}), ("not negative", {"scale": -0.5}),
    ("not negative", {"scale": math.inf}), ("fp16 or bf16", {"q_dtype": 2}), ("16-bit pages' type", {"format": 0, "q_dtype": 1}),
    ("NULL", {"q": None}), ("NULL", {"out": None}), ("NULL", {"lens": None}), ("bounds", {"bounds": None}),
    ("bounds", {"bounds": 0x1008}), ("aligned", {"q": {"data": 0x1008}}), ("aligned", {"out": 0x1008}),
    ("follow one another", {"q": {"stride_b": 512}}), ("workspace", {"ws": None}), ("workspace", {"ws_bytes": 16}),
    ("aligned", {"ws": 0x1004}), ("NULL table", {"table": None}), ("share memory", {"out": None})])
def test_sparse_refusals(c, word, kw):  # noqa: F811
    if word == "share memory":
        kw = {"out": c.at + 128}
    _refused(_sparse_call(c, **kw), c.lib, word)


@pytest.mark.parametrize("word,kw", [("negative", {"L": -1}), ("one position", {"pos": {"per_token": 1}}), ("one position", {"pos": None}),
                                     ("bounds", {"bounds": None}), ("bounds", {"bounds": 0x1008}), ("NULL table", {"table": None}),
                                     ("table shape", {"B": -1}), ("2^31 pages", {"B": 2 ** 30, "L": 10 ** 6, "n_table": 1024, "stride": 1024})])
def test_bounds_refusals(c, word, kw):  # noqa: F811
    a = dict(B=1, L=5, table=c.at, n_table=2, stride=2, pos={}, bounds=c.at, **{})
    a.update(kw)
    rc = c.lib.fkv_paged_bounds(R(c.pages()), a["bounds"], a["B"], a["L"], a["table"], a["n_table"], a["stride"],
                                None if a["pos"] is None else R(c.pos(**a["pos"])), None, None)
    _refused(rc, c.lib, word)


@pytest.mark.parametrize("word,kw", [
    ("65535", {"B": 65536}), ("65535", {"B": -1}), ("63", {"K": 64}), ("63", {"K": -1}), ("vocabulary", {"V": 0}),
    ("dtype", {"dtype": 3}), ("NULL", {"target": None}), ("NULL", {"draft": {"data": None}}), ("NULL", {"tokens": None}),
    ("NULL", {"uniforms": None}), ("NULL", {"out": None}), ("NULL", {"accepted": None}), ("workspace", {"ws": None}),
    ("workspace", {"ws": 0x1004}), ("workspace", {"ws_bytes": 15})])
def test_verify_refusals(c, word, kw):  # noqa: F811
    a = dict(target={}, draft={}, dtype=2, B=1, K=3, V=100, tokens=c.at, uniforms=c.at, out=c.at, accepted=c.at, ws=c.at, ws_bytes=1 << 30)
    a.update(kw)
    rows = [None if a[n] is None else R(c.rows(**a[n])) for n in ("target", "draft")]
    rc = c.lib.fkv_verify_drafts(*rows, a["dtype"], a["B"], a["K"], a["V"], a["tokens"], 1, a["uniforms"], None, a["out"],
                                 a["accepted"], a["ws"], a["ws_bytes"], None)
    _refused(rc, c.lib, word)


@pytest.mark.parametrize("word,kw", BAD_PAGES)
def test_page_refusals(c, word, kw):  # noqa: F811
    pg = c.pages(**kw)
    _refused(_rows_call(c, pg), c.lib, word)
    _refused(_sparse_call(c, pg), c.lib, word)
    _refused(c.lib.fkv_paged_attn_rows_workspace(R(pg), 2, 1, 3, 0, 16), c.lib, word)
    _refused(c.lib.fkv_paged_attn_sparse_workspace(R(pg), 2, 1, 4, 2, 16), c.lib, word)
    _refused(c.lib.fkv_paged_bounds(R(pg), c.at, 1, 5, c.at, 2, 2, R(c.pos()), None, None), c.lib, word)
    _refused(_rows_call(c, 0), c.lib, "NULL pages")
    _refused(_sparse_call(c, 0), c.lib, "NULL pages")


def test_empty_calls_do_nothing(c):  # noqa: F811
    pg = R(c.pages())
    assert _rows_call(c, B=0, q=None, out=None, ws=None) == 0 and _rows_call(c, L=0, q=None, out=None, ws=None) == 0
    assert _sparse_call(c, B=0, q=None, out=None, ws=None) == 0
    for B, L, n in ((0, 5, 2), (1, 0, 2), (1, 5, 0)):
        assert c.lib.fkv_paged_bounds(pg, c.at, B, L, c.at, n, n, R(c.pos()), None, None) == 0
    assert c.lib.fkv_verify_drafts(None, None, 0, 0, 3, 9, None, 0, None, None, None, None, None, 0, None) == 0


def test_workspaces(c):  # noqa: F811
    """Sizes are known without a device, and do not pass a few records for each
    row of the chip's workgroups."""
    for H, Hq, D in ((2, 4, 64), (8, 64, 128), (1, 40, 128)):
        pg = R(c.pages(H=H, D=D))
        for B in (1, 7, 64):
            for L, shared in ((1, 0), (4, 0), (1, 1024), (5, 65536), (500, 0)):
                for n in (0, 1, 128, 4096, 2 ** 17):
                    size = c.lib.fkv_paged_attn_rows_workspace(pg, Hq, B, L, shared, n)
                    assert 0 <= size <= max(1 << 28, B * Hq * L * 40 * 4 * (D + 4))
            assert 0 < c.lib.fkv_paged_attn_sparse_workspace(pg, Hq, B, 512, 64, 8192) <= 1 << 28
    assert c.lib.fkv_verify_drafts_workspace(64, 5, 128000) > 0


def test_compiled_calls_leave_what_is_not_plain():
    """Without a device every call is left to Python, whatever its arguments are."""
    calls = _lib.calls()
    x, i = torch.zeros(2, 2, 3, 64), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: calls.attend_tokens((0, 0), x, i[None], i, None, 0, None, None, False, None, 0),
                 lambda: calls.attend_tokens(), lambda: calls.attend_tokens(*[x] * 11), lambda: calls.attend_tokens(*[None] * 11),
                 lambda: calls.attend_sparse((0, 0), x, x, i[None], i, 3, None, 0, None, None, False, False),
                 lambda: calls.attend_sparse(), lambda: calls.attend_sparse(*[i] * 12),
                 lambda: calls.bound((0, 0), x, i[None], 0, 3, None), lambda: calls.bound(*[i] * 6),
                 lambda: calls.verify(x[0], None, i, x, None), lambda: calls.verify(), lambda: calls.verify(*[1] * 5)):
        assert call() is NotImplemented
