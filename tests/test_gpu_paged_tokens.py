"""Attention of several new tokens per sequence, and of sequences that begin
alike, against the 64-bit restatement: each query's own limit, padded batches,
beginnings in one sequence's pages, infinite and NaN rows that a query does not
attend to, strides, split rows, streams, captured graphs."""

import math

import numpy as np
import pytest
import torch

import _paged_ref as ref
from test_gpu_paged import DTYPES, FORMATS, _bits_equal, _filled, _flush, _randn, _spoil, _table

pytestmark = pytest.mark.gpu

KINDS = [("fp16", "fp16"), ("bf16", "bf16"), ("fp8", "fp16"), ("fp8", "bf16"), ("fp8_int4", "fp16"), ("fp8_int4", "bf16")]


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.load()
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _bound(out, spread, ds, n, fmt, dtype, mag):
    """What a result may be off by: its own rounding; each weight's relative
    error, from its score (twice, once in the sum), from exp2 (2^-22) and from its
    16-bit form (half a step of n bits is 2^-n): bf16 results one rounded bf16
    number, 2^-8; fp16 pages one fp16 number, 2^-11, or 2^-25 where it
    is small (the largest weight is 2^7 or more: 2^-32 of it, times the largest
    value); otherwise two bf16 numbers, the first cut off, which leaves less than 2^-7,
    and that rounded, 2^-15.  fp32 sums: of 32 tokens four products of 16,
    each rounded twice at most, then waves and workgroups."""
    n = max(int(n), 1)
    one = 2.0 ** -11 if fmt == "fp16" else 2.0 ** -8 if fmt != "fp16" and dtype == torch.bfloat16 else 2.0 ** -15
    rel = 2 * ds[..., None] * 1.01 + one + 2.0 ** -21 + (n / 4 + 64) * 2.0 ** -24
    return ref.UNIT[dtype] * np.abs(out) + ref.TINY[dtype] + rel * spread + n * 2.0 ** -32 * mag


def _values(layer):
    """As ``ref.page_values``; an INT4 value is scale (code - 8) + (min + 8 scale)
    here, and its error relative to the magnitudes of both."""
    k, v, mag = ref.page_values(layer)
    if layer.fmt == "fp8_int4":
        sz = ref.f64(layer.v_scale)
        with np.errstate(invalid="ignore"):
            shift = sz[..., 1:] + 8 * sz[..., :1]
            mag = np.abs(v - shift) + np.abs(shift)
    return k, v, mag


def _check(layer, q, table, lens, n_new=None, shared=0, scale=None, read_table=None, **kw):
    """attend_tokens against the restatement, by the table that the definition
    reads (``read_table``: the first row's pages where they are shared)."""
    B, Hq, L, D = q.shape
    out, lse = layer.attend_tokens(q, table.cuda(), _i32(lens), scale=scale, return_lse=True, shared=shared,
                                   n_new=None if n_new is None else _i32(n_new), **kw)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (B, Hq, L)
    s = D ** -0.5 if scale is None else scale
    t = (table if read_table is None else read_table).numpy()
    values, q64 = _values(layer), ref.f64(q)
    mag = max(1.0, float(np.nanmax(np.where(np.isfinite(values[1]), np.abs(values[1]), 0.0))))
    got, glse = ref.f64(out), ref.f64(lse)
    new = [L] * B if n_new is None else [min(max(n, 0), L) for n in n_new]
    have = [min(max(n + kw.get("lens_add", 0), 0), t.shape[1] * layer.page_size) for n in lens]
    for l in range(L):
        limit = [max(h - n + l + 1, 0) if l < n else 0 for h, n in zip(have, new)]
        want, wlse, spread, ds = ref.attend(q64[:, :, l], values, t, limit, layer.page_size, layer.n_pages, s)
        real = np.array([l < n for n in new])
        tol = _bound(want, spread, ds, max(limit), layer.fmt, q.dtype, mag)
        err = np.abs(got[:, :, l] - want)[real]
        assert (err <= tol[real]).all(), f"token {l}: {np.nanmax(err / tol[real])} of the bound, NaN {np.isnan(err).sum()}"
        none = np.isinf(wlse)
        assert (glse[:, :, l][none] == -np.inf).all()
        ltol = 2 * ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(np.where(none, 0.0, wlse))
        assert (np.abs(glse[:, :, l][~none] - wlse[~none]) <= ltol[~none]).all()
        if "out" not in kw:
            assert (got[:, :, l][~real] == 0).all()
    return out


EDGES = [0, 1, 3, 15, 17, 33, 127, 128, 130, 300]


@pytest.mark.parametrize("fmt,qd", KINDS)
@pytest.mark.parametrize("D,H,G,page,L", [(128, 2, 4, 16, 5), (64, 2, 7, 32, 4), (128, 1, 1, 64, 1), (64, 1, 3, 16, 33),
                                          (128, 1, 8, 128, 19), (64, 1, 40, 32, 2)])
def test_edges(paged, fmt, qd, D, H, G, page, L):
    """Lengths around every border, shorter than the new tokens among them;
    one to eight waves' rows."""
    _flush("tokens", fmt, qd, D, H, G, page, L)
    counts = [-(-n // page) for n in EDGES]
    layer = _filled(paged, fmt, sum(counts) + 2, H, D, page, 20)
    table = _table(21, sum(counts) + 2, counts)
    _spoil(layer, table, EDGES)
    q = _randn(22, len(EDGES), L, H * G, D).to(DTYPES[qd]).cuda().transpose(1, 2)
    out = _check(layer, q, table, EDGES)
    assert bool((out[0] == 0).all())
    n_new = [(3 * b) % (L + 2) for b in range(len(EDGES))]  # (some more than there are)
    n_new[3] = -1
    _check(layer, q, table, EDGES, n_new)
    _check(layer, q, table, [n - 2 for n in EDGES], n_new, lens_add=2, scale=-0.05)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,H,G,L,lens", [(128, 1, 5, 3, [5003]), (64, 2, 4, 70, [900, 77, 2100]),
                                          (128, 1, 2, 300, [301, 1000]), (128, 2, 4, 2, [400] * 40)])
def test_split_rows(paged, fmt, D, H, G, L, lens):
    """Rows over several workgroups and workgroups of several rows; the same
    bits again, and with a bound that the lengths pass."""
    _flush("split", fmt, D, H, G, L)
    page = 32
    counts = [-(-n // page) for n in lens]
    layer = _filled(paged, fmt, sum(counts), H, D, page, 30, gain=2.0)
    table = _table(31, sum(counts), counts)
    q = (_randn(32, len(lens), H * G, L, D) * 3).to(DTYPES.get(fmt, torch.bfloat16)).cuda()
    a = _check(layer, q, table, lens)
    b = _check(layer, q, table, lens, max_len=max(lens))
    _check(layer, q, table, lens, max_len=1)
    for _ in range(3):
        _bits_equal(_check(layer, q, table, lens), a, "again")
        _bits_equal(layer.attend_tokens(q, table.cuda(), _i32(lens), max(lens)), b, "again")


UNEVEN = {
    "one long": [2900] + [3] * 8,
    "long last": [1] * 30 + [2500],
    "falling": [1900 - 190 * i for i in range(11)],
    "none": [0] * 7,
    "some none": [0, 1100, 0, 0, 700, 0, 64, 65],
    "many": [(97 * i * i) % 400 for i in range(130)],
}


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("name", UNEVEN)
@pytest.mark.parametrize("H", [1, 3])
def test_parts_of_uneven_sequences(paged, fmt, name, H):
    """Parts that the device makes of the lengths; a bound of the lengths that is
    too small or too large; padded batches."""
    lens = UNEVEN[name]
    B, D, G, L, page = len(lens), 64, 2, 3, 16
    _flush("uneven", fmt, name, H)
    counts = [max(1, -(-n // page)) for n in lens]
    layer = _filled(paged, fmt, sum(counts) + 2, H, D, page, 50)
    table = _table(51, sum(counts) + 2, counts)
    _spoil(layer, table, lens)
    q = _randn(52, B, H * G, L, D).to(DTYPES["bf16"]).cuda()
    for kw in ({}, {"max_len": max(lens)}, {"max_len": max(lens) // 3}, {"lens_add": -40}):
        _check(layer, q, table, lens, **kw)
    _check(layer, q, table, lens, [(2 * b) % (L + 1) for b in range(B)])
    # a captured call follows the lengths of its replays
    long, new = _i32(lens), torch.cuda.CUDAGraph()
    on = table.cuda()
    layer.attend_tokens(q, on, long)
    with torch.cuda.graph(new):
        out = layer.attend_tokens(q, on, long)
    for shift in (1, 3, 5):
        long.copy_(_i32([max(0, n - 170 * shift) for n in lens]))
        new.replay()
        _bits_equal(out.clone(), layer.attend_tokens(q, on, long), shift)


@pytest.mark.parametrize("fmt,qd", KINDS)
@pytest.mark.parametrize("D,H,G,L,B,shared", [(128, 2, 4, 1, 9, 256), (64, 1, 7, 3, 5, 48), (128, 1, 2, 2, 70, 1024),
                                              (64, 2, 1, 9, 2, 16), (64, 1, 4, 1, 150, 512), (64, 1, 4, 70, 4, 256)])
def test_shared_beginning(paged, fmt, qd, D, H, G, L, B, shared):
    """A beginning that all sequences share, read from the first row alone;
    sequences that end before it does, and with it."""
    _flush("shared", fmt, qd, D, H, G, L, B, shared)
    page = 16
    own = [(37 * b) % 90 for b in range(B)]
    lens = [shared + n for n in own]
    lens[1] = shared - 7
    if B > 4:
        lens[2], lens[4] = 0, shared
    n_shared, counts = shared // page, [-(-n // page) for n in own]
    n_pages = n_shared + sum(counts)
    layer = _filled(paged, fmt, n_pages, H, D, page, 50)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(51)).int()
    table = torch.full((B, n_shared + max(counts)), 2 ** 31 - 1, dtype=torch.int32)
    table[:, :n_shared] = order[:n_shared]
    at = n_shared
    for b, n in enumerate(counts):
        table[b, n_shared:n_shared + n] = order[at:at + n]
        at += n
    _spoil(layer, table, [max(n, shared) for n in lens])
    q = _randn(52, B, L, H * G, D).to(DTYPES[qd]).cuda().transpose(1, 2)
    elsewhere = table.clone()
    elsewhere[1:, :n_shared] = -5  # (not looked at)
    out = _check(layer, q, elsewhere, lens, shared=shared, read_table=table)
    _bits_equal(layer.attend_tokens(q, table.cuda(), _i32(lens), shared=shared), out, "the same table throughout")
    n_new = [(2 * b) % (L + 1) for b in range(B)]
    _check(layer, q, elsewhere, lens, n_new, shared=shared, read_table=table, max_len=max(lens))
    _check(layer, q, table, lens, shared=page)
    # one sequence shares with nobody
    _check(layer, q[:1], table[:1], lens[:1], shared=shared)


def test_all_of_the_tokens_shared(paged):
    layer = _filled(paged, "bf16", 8, 1, 128, 16, 55)
    table = torch.arange(8, dtype=torch.int32).view(1, 8).expand(3, -1).contiguous()
    q = _randn(56, 3, 4, 2, 128).bfloat16().cuda()
    _check(layer, q, table, [128, 127, 100], shared=128)
    _check(layer, q, table, [128, 127, 100], shared=112, n_new=[2, 0, 1])


@pytest.mark.parametrize("fmt,qd", KINDS)
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_rows_that_a_query_does_not_attend_to(paged, fmt, qd, bad):
    """Infinite and NaN keys and values of later tokens leave earlier queries as
    they are, and reach the later ones."""
    _flush("later", fmt, qd, bad)
    page, H, G, D, L = 16, 1, 3, 128, 6
    lens = [40, 133, 6]
    counts = [-(-n // page) for n in lens]
    layer = _filled(paged, fmt, sum(counts), H, D, page, 60)
    table = _table(61, sum(counts), counts)
    q = _randn(62, 3, H * G, L, D).to(DTYPES[qd]).cuda()
    want = layer.attend_tokens(q, table.cuda(), _i32(lens))
    hit = 3  # the new token with the bad rows
    for part in ("k", "v"):
        for b, n in enumerate(lens):
            p = n - L + hit
            at = (int(table[b, p // page]), 0, p % page)
            kept = {name: getattr(layer, name)[at].clone() for name in ("k", "v", "k_exp", "v_scale")
                    if getattr(layer, name) is not None}
            if layer.k_exp is None:
                getattr(layer, part)[at][5] = bad
            elif part == "k":
                layer.k[at][5] = 127  # (the NaN code)
            elif fmt == "fp8":
                layer.v[at][5] = 127
            else:
                layer.v_scale[at][1] = bad
            got = layer.attend_tokens(q, table.cuda(), _i32(lens))
            _bits_equal(got[b, :, :hit], want[b, :, :hit], f"{part} of sequence {b}, before")
            others = [i for i in range(3) if i != b]
            _bits_equal(got[others], want[others], "other sequences")
            after = got[b, :, hit:].float()
            if part == "v" and fmt != "fp8_int4":
                assert not bool(torch.isfinite(after[..., 5]).any())
                _bits_equal(after[..., :5], want[b, :, hit:, :5].float(), "other dims")
            elif part == "v":
                assert not bool(torch.isfinite(after).any())
            elif layer.k_exp is not None or math.isnan(bad):
                assert bool(torch.isnan(after).all())
            for name, t in kept.items():
                getattr(layer, name)[at] = t
    _bits_equal(layer.attend_tokens(q, table.cuda(), _i32(lens)), want, "restored")


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_outside_the_pool(paged, fmt):
    page, H, G, D, L = 16, 2, 3, 64, 4
    layer = _filled(paged, fmt, 30, H, D, page, 40)
    table = _table(41, 30, [10, 10, 10])
    table[0, 3], table[0, 9], table[1, 0], table[2, :] = -1, 30, 2 ** 30, -7
    q = _randn(42, 3, H * G, L, D).to(DTYPES.get(fmt, torch.float16)).cuda()
    out = _check(layer, q, table, [160, 10 ** 6, 100])
    assert bool((out[2] == 0).all())
    _check(layer, q, table, [-3, -2 ** 31, 0])
    both = table.clone()
    both[1:, :4] = table[0, :4]
    _check(layer, q, table, [160, 100, 61], shared=64, read_table=both)


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_token_far_above_the_others(paged, fmt):
    """One token 16 powers of two above the others, of value zero: the others'
    weights are what the result is made of."""
    page, D, n = 16, 128, 200
    layer = paged.PagedLayer(13, 1, D, page, fmt)
    k = torch.zeros(1, 1, n, D)
    k[0, 0, 77, 0] = 16.0
    v = _randn(71, 1, 1, n, D)
    v[0, 0, 77] = 0.0
    table = torch.arange(13, dtype=torch.int32).view(1, 13)
    layer.write(k.cuda(), v.cuda(), table.cuda(), 0)
    q = torch.zeros(1, 4, 3, D)
    q[..., 0] = 1.0
    q = q.to(DTYPES.get(fmt, torch.float16)).cuda()
    _check(layer, q, table, [n], scale=math.log(2.0))
    _check(layer, q.expand(2, -1, -1, -1), table.expand(2, -1), [n, n - 5], shared=96, scale=math.log(2.0))


def test_scores_at_the_edge_of_fp32(paged):
    layer = paged.PagedLayer(20, 1, 64, 16, "bf16")
    layer.k.fill_(0.0)
    layer.k[..., 0] = -1.0e18
    layer.v.copy_(_randn(65, 20, 1, 16, 64))
    table = torch.arange(20, dtype=torch.int32).view(1, 20)
    q = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0e18
    _check(layer, q, table, [300], scale=128.0)


def test_strides_results_and_copies(paged):
    layer = _filled(paged, "fp8", 24, 2, 64, 16, 80)
    table = _table(81, 24, [12, 12])
    lens, new = [190, 100], [4, 2]
    q = _randn(82, 2, 4, 6, 64).half().cuda().transpose(1, 2)  # (2, 6, 4, 64), tokens before heads
    want = _check(layer, q, table, lens)
    assert want.stride() == q.stride()
    padded = _check(layer, q, table, lens, new)
    for out in (torch.full((2, 6, 4, 64), 7.0, dtype=torch.float16, device="cuda"),
                torch.full((2, 4, 6, 64), 7.0, dtype=torch.float16, device="cuda").transpose(1, 2),
                torch.full((2, 6, 4, 128), 7.0, dtype=torch.float16, device="cuda")[..., ::2],
                torch.full((2 * 6 * 4 * 64 + 1,), 7.0, dtype=torch.float16, device="cuda")[1:].view(2, 6, 4, 64)):
        assert layer.attend_tokens(q, table.cuda(), _i32(lens), out=out) is out
        _bits_equal(out, want, "out")
        out.fill_(7.0)
        layer.attend_tokens(q, table.cuda(), _i32(lens), out=out, n_new=_i32(new))
        assert bool((out[1, :, 2:] == 7.0).all())
        _bits_equal(out[1, :, :2], padded[1, :, :2], "real tokens")
        _bits_equal(out[0], padded[0], "real tokens")
    x = q.clone()
    assert layer.attend_tokens(x, table.cuda(), _i32(lens), out=x) is x
    _bits_equal(x, want, "in place")
    odd = torch.zeros(2 * 6 * 4 * 64 + 3, dtype=torch.float16, device="cuda")[3:].view(2, 6, 4, 64)
    odd.copy_(q)
    _bits_equal(layer.attend_tokens(odd, table.cuda(), _i32(lens)), want, "unaligned query")
    wide = torch.zeros(2, 24, dtype=torch.int32)
    wide[:, ::2] = table
    _bits_equal(layer.attend_tokens(q, wide.cuda()[:, ::2], _i32(lens)), want, "strided table")
    one = q[:, :, :1]
    _bits_equal(layer.attend_tokens(one.expand(-1, -1, 3, -1), table.cuda(), _i32(lens))[:, :, 2],
                layer.attend_tokens(one, table.cuda(), _i32(lens))[:, :, 0], "one query for three tokens")


def test_refusals(paged):
    layer = paged.PagedLayer(4, 2, 64, 16, "fp16")
    table = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    lens, q = _i32([3, 3]), torch.zeros(2, 4, 3, 64, dtype=torch.float16, device="cuda")
    from foveated_kv_amd._lib import FkvLibraryError

    bad = [
        (ValueError, lambda: layer.attend_tokens(q[:, :3], table, lens)),
        (ValueError, lambda: layer.attend_tokens(q[..., :32], table, lens)),
        (ValueError, lambda: layer.attend_tokens(q[0], table, lens)),
        (TypeError, lambda: layer.attend_tokens(q.float(), table, lens)),
        (TypeError, lambda: layer.attend_tokens(q.bfloat16(), table, lens)),
        (TypeError, lambda: layer.attend_tokens(None, table, lens)),
        (ValueError, lambda: layer.attend_tokens(q, table[:1], lens)),
        (TypeError, lambda: layer.attend_tokens(q, table, lens.long())),
        (TypeError, lambda: layer.attend_tokens(q, table, lens, n_new=lens.long())),
        (TypeError, lambda: layer.attend_tokens(q, table, lens, n_new=lens[:1])),
        (ValueError, lambda: layer.attend_tokens(q, table, lens, shared=15)),
        (ValueError, lambda: layer.attend_tokens(q, table, lens, shared=-16)),
        (ValueError, lambda: layer.attend_tokens(q, table, lens, shared=48)),
        (TypeError, lambda: layer.attend_tokens(q, table, lens, shared=16.0)),
        (ValueError, lambda: layer.attend_tokens(q, table, lens, lens_add=2 ** 31)),
        (ValueError, lambda: layer.attend_tokens(q, table, lens, out=q.float())),
        (ValueError, lambda: layer.attend_tokens(q, table, lens, out=q[:, :, :1].expand(-1, -1, 3, -1))),
        (FkvLibraryError, lambda: layer.attend_tokens(q, table, lens, out=q.as_strided(q.shape, (768, 64, 64, 1)))),
        (FkvLibraryError, lambda: layer.attend_tokens(q[:1], table[:1], lens[:1], out=q.flatten()[64:64 + 768].view(1, 4, 3, 64))),
        (FkvLibraryError, lambda: layer.attend_tokens(q, table, lens, scale=float("nan"))),
        (RuntimeError, lambda: layer.attend_tokens(q.clone().requires_grad_(), table, lens)),
        (ValueError, lambda: layer.attend(q, table, lens)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("accepted", i)
    assert layer.attend_tokens(q[:0], table[:0], lens[:0]).shape == (0, 4, 3, 64)
    assert layer.attend_tokens(q[:, :, :0], table, lens).shape == (2, 4, 0, 64)
    assert bool((layer.attend_tokens(q, table[:, :0], lens) == 0).all())


def test_far_offsets(paged):
    """Pages that lie past 2^31 bytes and elements of the pool."""
    page, H, D, n_pages = 64, 8, 128, 36000
    layer = paged.PagedLayer(n_pages, H, D, page, "fp8")
    small = paged.PagedLayer(3, H, D, page, "fp8")
    far = torch.tensor([[n_pages - 1, 0, n_pages - 2]] * 2, dtype=torch.int32).cuda()
    near = torch.tensor([[2, 0, 1]] * 2, dtype=torch.int32).cuda()
    k, v = (_randn(80 + i, 1, H, 3 * page, D).bfloat16().cuda() for i in range(2))
    layer.write(k, v, far[:1], 0)
    small.write(k, v, near[:1], 0)
    q, lens = _randn(82, 2, 32, 4, D).bfloat16().cuda(), _i32([3 * page - 1, 150])
    for shared in (0, 128):
        _bits_equal(layer.attend_tokens(q, far, lens, shared=shared), small.attend_tokens(q, near, lens, shared=shared), "far")


@pytest.mark.parametrize("fmt", ["bf16", "fp8_int4"])
def test_captured_on_two_streams(paged, fmt):
    """Steps of three drafted tokens over a shared beginning, captured once for
    each of two caches and replayed side by side while both grow and the numbers
    of real tokens change: the eager result's bits."""
    _flush("graphs", fmt)
    page, H, G, D, B, L, steps, shared = 16, 2, 4, 128, 3, 3, 25, 32

    def cache(seed):
        layer = _filled(paged, fmt, 62, H, D, page, seed)
        table = _table(seed + 1, 62, [20, 20, 20])
        table[1:, :2] = table[0, :2]
        xs = [(_randn(seed + 10 + i, B, H, L, D).bfloat16().cuda(), _randn(seed + 100 + i, B, H, L, D).bfloat16().cuda(),
               _randn(seed + 200 + i, B, H * G, L, D).bfloat16().cuda(), _i32([i % 4, (i + 1) % 4, 3])) for i in range(steps)]
        return layer, table.cuda(), _i32([100, 40, 200]), xs

    def step(layer, table, start, k, v, q, new):
        layer.write(k, v, table, start, n_new=new)
        return layer.attend_tokens(q, table, start + new, n_new=new, shared=shared)

    eager = []
    for seed in (300, 700):
        layer, table, start, xs = cache(seed)
        eager.append([])
        for x in xs:
            eager[-1].append(step(layer, table, start, *x).clone())
            start.add_(x[3])
    torch.cuda.synchronize()
    runs = []
    for seed in (300, 700):
        layer, table, start, xs = cache(seed)
        bufs = [t.clone() for t in xs[0]]
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            out = step(layer, table, start, *bufs)
        runs.append((g, s, bufs, out, start, xs, layer, table))
    torch.cuda.synchronize()
    for i in range(steps):
        for g, s, bufs, out, start, xs, *_ in runs:
            with torch.cuda.stream(s):
                for dst, src in zip(bufs, xs[i]):
                    dst.copy_(src)
                g.replay()
                start.add_(xs[i][3])
        if i % 7 == 3:
            torch.cuda.synchronize()
            torch.randn(1000, device="cuda").sum().item()
        for (g, s, bufs, out, *_), want in zip(runs, eager):
            s.synchronize()
            _bits_equal(out, want[i], f"replay {i}")
