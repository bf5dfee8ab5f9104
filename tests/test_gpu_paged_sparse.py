"""Bounds of pages, the choice of pages by them and the attention over these,
against 64-bit restatements: the bounds' bits, the pages exactly, equal scores,
lengths around every border, pages outside the pool, captured graphs."""

import math

import numpy as np
import pytest
import torch

import _paged_ref as ref
from test_gpu_paged import DTYPES, FORMATS, _bits_equal, _filled, _flush, _randn, _spoil, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.load()
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _with_bounds(paged, layer):
    b = torch.full((layer.n_pages, layer.n_kv_heads, 2, layer.head_dim), 77.0, dtype=torch.bfloat16, device="cuda")
    return paged.PagedLayer.wrap(layer.fmt, layer.k, layer.v, layer.k_exp, layer.v_scale, bounds=b)


def _outward(x, up):
    """float64 (of fp32 numbers) -> bf16 numbers as float64: a search over the
    neighbours of the rounded one."""
    t = torch.from_numpy(np.asarray(x)).float()
    r = t.bfloat16()
    step = torch.nextafter(r, torch.full_like(r, math.inf if up else -math.inf))
    bad = (r.float() < t) if up else (r.float() > t)
    return torch.where(bad, step, r)


def _want_bounds(layer, before, table, first, last):
    """Bounds after tokens [first, last) of each sequence were bounded."""
    out, keys, page = before.clone().cpu(), ref.page_values(layer)[0], layer.page_size
    for b, (f, n) in enumerate(zip(first, last)):
        f, n = max(f, 0), min(n, table.shape[1] * page)
        for i in range(f // page, -(-n // page) if n > f else 0):
            pid = int(table[b, i])
            if 0 <= pid < layer.n_pages:
                k = keys[pid][:, :min(page, n - i * page)]
                lo, hi = np.nanmin(k, 1), np.nanmax(k, 1)
                out[pid, :, 0], out[pid, :, 1] = _outward(lo, False), _outward(hi, True)
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,H,page", [(128, 2, 16), (64, 3, 32), (128, 1, 64), (64, 2, 256)])
def test_bounds(paged, fmt, D, H, page):
    _flush("bounds", fmt, D, H, page)
    layer = _with_bounds(paged, _filled(paged, fmt, 21, H, D, page, 10))
    table = _table(11, 21, [5, 5, 5, 5])
    table[2, 1], table[3, 4] = -1, 21
    before = layer.bounds.clone()
    start, n = [0, page - 1, page + 3, 4 * page - 2], 2 * page + 1
    new = [2 * page + 1, 0, 5, 2 * page + 1]
    layer.bound(table.cuda(), torch.tensor(start).cuda(), n, n_new=_i32(new))
    want = _want_bounds(layer, before, table, start, [s + m for s, m in zip(start, new)])
    _bits_equal(layer.bounds, want, "bounds")
    layer.bound(table.cuda(), 3, n)
    _bits_equal(layer.bounds, _want_bounds(layer, want, table, [3] * 4, [3 + n] * 4), "one start for all")
    layer.bound(table.cuda(), torch.tensor([-40, 5 * page, 6 * page, 0]).cuda(), 33)
    layer.bound(table.cuda(), 0, 0)
    layer.bound(table[:0].cuda(), 0, 5)


def test_bounds_of_special_keys(paged):
    """Infinities, NaN, zeros of either sign, numbers between those of bf16."""
    layer = _with_bounds(paged, paged.PagedLayer(1, 1, 64, 16, "fp16"))
    layer.k.fill_(0.0)
    k = layer.k[0, 0]
    k[3, 0], k[4, 1], k[5, 2] = math.inf, -math.inf, math.nan
    k[:, 3] = math.nan
    k[:, 4] = 1.0009765625  # 1 + 2^-10
    k[:, 5] = -1.0009765625
    k[:, 6] = 65504.0
    k[:, 7] = 2.0 ** -24
    layer.bound(_i32([[0]]), 0, 16)
    lo, hi = layer.bounds[0, 0].float().cpu()
    assert hi[0] == math.inf and lo[0] == 0 and lo[1] == -math.inf and hi[1] == 0 and lo[2] == hi[2] == 0
    assert lo[3] == math.inf and hi[3] == -math.inf  # (no key)
    assert lo[4] == 1.0 and hi[4] == 1.0078125 and lo[5] == -1.0078125 and hi[5] == -1.0
    assert lo[6] == 65280.0 and hi[6] == 65536.0 and lo[7] == hi[7] == 2.0 ** -24


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_keeps_the_bounds(paged, fmt):
    """Steps, chunks, padded batches and tokens taken back and written again."""
    page, H, D, B = 16, 2, 64, 3
    layer = paged.PagedLayer(12, H, D, page, fmt, bounds=True)
    table = _table(15, 12, [4, 4, 4])
    rope = paged.Rope(D, max_positions=64)
    lens, want = [0] * B, layer.bounds.clone().cpu()
    for i, (L, new, back) in enumerate([(20, [20, 3, 17], [0, 0, 0]), (1, [1, 1, 1], [0, 0, 0]), (5, [5, 0, 2], [3, 2, 0]),
                                        (1, [1, 1, 1], [0, 0, 9]), (16, [16, 16, 16], [0, 0, 0])]):
        lens = [n - x for n, x in zip(lens, back)]
        k, v = _randn(16 + i, B, H, L, D).cuda(), _randn(30 + i, B, H, L, D).cuda()
        layer.write(k, v, table.cuda(), _i32(lens), n_new=_i32(new) if i != 1 else None, rope=rope)
        want = _want_bounds(layer, want, table, lens, [n + m for n, m in zip(lens, new)])
        lens = [n + m for n, m in zip(lens, new)]
        _bits_equal(layer.bounds, want, f"write {i}")


def _want_pages(layer, q, table, lens, n_select):
    """The pages of each sequence and KV head, from the bounds in 64 bits."""
    B, Hq = q.shape[:2]
    H, page = layer.n_kv_heads, layer.page_size
    box, q64 = ref.f64(layer.bounds), ref.f64(q)[:, :, 0].reshape(B, H, Hq // H, -1)
    out = np.full((B, H, n_select), -1, dtype=np.int64)
    for b in range(B):
        count = -(-min(max(lens[b], 0), table.shape[1] * page) // page)
        for h in range(H):
            score = []
            for i in range(count - 1):
                pid = int(table[b, i])
                if not 0 <= pid < layer.n_pages:
                    score.append(-math.inf)
                    continue
                with np.errstate(invalid="ignore"):
                    lo, hi = np.minimum(q64[b, h], 0) * box[pid, h, 0], np.maximum(q64[b, h], 0) * box[pid, h, 1]
                    s = lo.sum(-1) + hi.sum(-1)
                score.append(np.where(np.isnan(s), math.inf, s).max())
            best = sorted(range(count - 1), key=lambda i: (-score[i], i))[:n_select - 1]
            picked = sorted(best) + ([count - 1] if count else [])
            out[b, h, :len(picked)] = picked
    return out


def _check(layer, q, table, lens, n_select, scale=None, **kw):
    out, lse, pages = layer.attend_sparse(q, table.cuda(), _i32(lens), n_select, scale=scale, return_lse=True, return_pages=True, **kw)
    B, Hq, _, D = q.shape
    H, page = layer.n_kv_heads, layer.page_size
    G = Hq // H
    assert out.shape == q.shape and lse.shape == (B, Hq) and pages.shape == (B, H, n_select)
    have = [min(max(n + kw.get("lens_add", 0), 0), table.shape[1] * page) for n in lens]
    picked = _want_pages(layer, q, table, have, n_select)
    assert np.array_equal(pages.cpu().numpy(), picked)
    s = D ** -0.5 if scale is None else scale
    values, q64 = ref.page_values(layer), ref.f64(q)[:, :, 0]
    for h in range(H):
        # each head's own table and length
        t = np.where(picked[:, h] >= 0, np.take_along_axis(table.numpy().astype(np.int64), np.maximum(picked[:, h], 0), 1)
                     if table.shape[1] else -1, -1)
        n = [0 if m == 0 else ((picked[b, h] >= 0).sum() - 1) * page + m - (m - 1) // page * page for b, m in enumerate(have)]
        mine = [v[:, h:h + 1] for v in values]
        want, wlse, spread, ds = ref.attend(q64[:, h * G:(h + 1) * G], mine, t, n, page, layer.n_pages, s)
        tol = ref.attend_bound(want, spread, ds, n, q.dtype)
        err = np.abs(ref.f64(out)[:, h * G:(h + 1) * G, 0] - want)
        assert (err <= tol).all(), f"error {np.nanmax(err / tol)} of the bound, NaN {np.isnan(err).sum()}"
        none, g = np.isinf(wlse), ref.f64(lse)[:, h * G:(h + 1) * G]
        assert (g[none] == -np.inf).all()
        ltol = 2 * ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(np.where(none, 0.0, wlse))
        assert (np.abs(g[~none] - wlse[~none]) <= ltol[~none]).all()
    return out


LENS = [0, 1, 16, 17, 300, 641, 640, 2000]


@pytest.mark.parametrize("fmt,qd", [("fp16", "fp16"), ("bf16", "bf16"), ("fp8", "fp16"), ("fp8", "bf16"), ("fp8_int4", "fp16"),
                                    ("fp8_int4", "bf16")])
@pytest.mark.parametrize("D,H,G,page", [(128, 2, 4, 16), (64, 3, 7, 32), (128, 1, 33, 64), (64, 1, 1, 16)])
def test_attend_sparse(paged, fmt, qd, D, H, G, page):
    _flush("sparse", fmt, qd, D, H, G, page)
    counts = [-(-n // page) for n in LENS]
    layer = _with_bounds(paged, _filled(paged, fmt, sum(counts) + 2, H, D, page, 20))
    table = _table(21, sum(counts) + 2, counts)
    layer.bound(table.cuda(), 0, max(LENS), n_new=_i32(LENS))
    _spoil(layer, table, LENS)
    q = _randn(22, len(LENS), 1, H * G, D).to(DTYPES[qd]).cuda().transpose(1, 2)
    for n_select in (1, 2, 7, 10, 64, max(counts), max(counts) + 5):
        out = _check(layer, q, table, LENS, n_select)
        assert bool((out[0] == 0).all())
    _check(layer, q, table, [n - 1 for n in LENS], 5, lens_add=1, max_len=max(LENS), scale=0.3)
    _check(layer, q, table, LENS, 5, max_len=10)


def test_equal_scores_go_to_the_lower_page(paged):
    """Pages with the same keys, more than a workgroup has threads; scores
    that differ in their last bits alone."""
    page, D, n = 16, 64, 2600
    layer = _with_bounds(paged, paged.PagedLayer(n, 1, D, page, "bf16"))
    layer.k.fill_(0.25)
    layer.v.copy_(_randn(30, n, 1, page, D))
    table = torch.randperm(n, generator=torch.Generator().manual_seed(31)).int().view(1, n)
    for i in (7, 1500, 2400):
        layer.k[int(table[0, i])] = 0.5
    layer.k[int(table[0, 40])] = -3.0
    layer.k[int(table[0, 100]), :, 0, 5] = 0.251953125  # (the next bf16 number)
    layer.bound(table.cuda(), 0, n * page)
    q = torch.ones(1, 2, 1, D, dtype=torch.bfloat16, device="cuda")
    q[0, 1] = 0.5
    for k in (1, 2, 4, 5, 6, 30, 1030, 2599, 2600):
        _check(layer, q, table, [n * page], k)
    pages = layer.attend_sparse(q, table.cuda(), _i32([n * page]), 7, return_pages=True)[1]
    assert pages.flatten().tolist() == [0, 1, 7, 100, 1500, 2400, 2599]


def test_scores_that_fp32_cannot_tell_apart(paged):
    """Bounds whose difference is 2^-30 of them, in either order."""
    page, D = 16, 64
    layer = _with_bounds(paged, paged.PagedLayer(6, 1, D, page, "bf16"))
    layer.k.fill_(0.0)
    layer.k[..., 0] = 256.0
    for i, x in enumerate([0.0, 2.0 ** -22, 2.0 ** -24, 2.0 ** -21, 2.0 ** -23]):
        layer.k[i, ..., 1] = x
    table = torch.arange(6, dtype=torch.int32).view(1, 6)
    layer.bound(table.cuda(), 0, 6 * page)
    q = torch.ones(1, 1, 1, D, dtype=torch.bfloat16, device="cuda")
    for k, want in ((2, [3, 5]), (3, [1, 3, 5]), (4, [1, 3, 4, 5]), (5, [1, 2, 3, 4, 5])):
        assert layer.attend_sparse(q, table.cuda(), _i32([6 * page]), k, return_pages=True)[1].flatten().tolist() == want


@pytest.mark.parametrize("qd", [torch.bfloat16, torch.float16])
def test_long_contexts(paged, qd):
    """More pages than the choice holds keys of (8192), scores of all kinds: far
    apart, near one another, and equal."""
    page, D, n = 16, 64, 9001
    layer = _with_bounds(paged, paged.PagedLayer(600, 1, D, page, "fp8"))
    k = _randn(50, 600, 1, page, D)
    k[200:400] = k[200] + 1e-3 * _randn(51, 200, 1, page, D)
    k[400:] *= 0.01
    ids = torch.arange(600, dtype=torch.int32, device="cuda").view(600, 1)
    layer.write(k.cuda(), _randn(52, 600, 1, page, D).cuda(), ids, 0)
    table = torch.randint(0, 600, (1, n), generator=torch.Generator().manual_seed(53)).int()
    q = _randn(54, 1, 3, 1, D).to(qd).cuda()
    for k in (2, 40, 700, 3500):
        _check(layer, q, table, [n * page - 3], k)
    assert n > 8192


def test_very_long_context(paged):
    """More pages than the choice has marks for (2^18), of which many are equal."""
    page, D, n = 16, 64, 2 ** 18 + 1000
    layer = _with_bounds(paged, paged.PagedLayer(50, 1, D, page, "bf16"))
    layer.k.copy_(_randn(55, 50, 1, page, D))
    layer.v.copy_(_randn(56, 50, 1, page, D))
    layer.bound(torch.arange(50, dtype=torch.int32, device="cuda").view(50, 1), 0, page)
    table = torch.randint(0, 50, (1, n), generator=torch.Generator().manual_seed(57)).int()
    q = _randn(58, 1, 1, 1, D).bfloat16().cuda()
    for k in (3, 6000):
        _check(layer, q, table, [n * page], k)


def test_scores_that_overflow_fp32(paged):
    """Bounds whose products pass the end of fp32's range, of either sign."""
    page, D = 16, 64
    layer = _with_bounds(paged, paged.PagedLayer(8, 1, D, page, "bf16"))
    layer.k.fill_(1.0)
    for i, x in enumerate([3e38, -3e38, 2e38, 1.0, -1e38, 2.5e38, 1e30]):
        layer.k[i, ..., :3] = x
    layer.bound(torch.arange(8, dtype=torch.int32, device="cuda").view(8, 1), 0, page)
    table = torch.arange(8, dtype=torch.int32).view(1, 8)
    q = torch.full((1, 2, 1, D), 4.0, dtype=torch.bfloat16, device="cuda")
    for k, want in ((2, [0, 7]), (3, [0, 5, 7]), (4, [0, 2, 5, 7]), (6, [0, 2, 3, 5, 6, 7]), (7, [0, 2, 3, 4, 5, 6, 7])):
        got = layer.attend_sparse(q, table.cuda(), _i32([8 * page]), k, return_pages=True, scale=0.0)[1]
        assert got.flatten().tolist() == want


def test_pages_outside_the_pool_and_bounds_not_finite(paged):
    page, H, G, D = 16, 2, 3, 64
    layer = _with_bounds(paged, _filled(paged, "bf16", 30, H, D, page, 40))
    table = _table(41, 30, [10, 10, 10])
    layer.bound(table.cuda(), 0, 160)
    table[0, 3], table[0, 9], table[1, 0], table[2, :] = -1, 30, 2 ** 30, -7
    layer.bounds[int(table[1, 5]), 0, 1, 9] = math.inf
    layer.bounds[int(table[1, 6]), 1, 0, 9] = math.nan
    q = _randn(42, 3, H * G, 1, D).bfloat16().cuda()
    q[1, 0, 0, 9] = 0.0
    for k in (2, 4, 9, 12):
        out = _check(layer, q, table, [160, 10 ** 6, 100], k)
        assert bool((out[2] == 0).all())
    _check(layer, q, table, [-3, -2 ** 31, 0], 3)


def test_refusals(paged):
    from foveated_kv_amd._lib import FkvLibraryError

    plain = paged.PagedLayer(4, 2, 64, 16, "fp16")
    layer = paged.PagedLayer(4, 2, 64, 16, "fp16", bounds=True)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), _i32([3])
    q = torch.zeros(1, 4, 1, 64, dtype=torch.float16, device="cuda")
    bad = [
        (ValueError, lambda: plain.attend_sparse(q, table, lens, 2)),
        (ValueError, lambda: plain.bound(table, 0, 3)),
        (ValueError, lambda: layer.attend_sparse(q, table, lens, 0)),
        (TypeError, lambda: layer.attend_sparse(q, table, lens, 1.5)),
        (ValueError, lambda: layer.attend_sparse(q.expand(-1, -1, 2, -1), table, lens, 2)),
        (TypeError, lambda: layer.attend_sparse(q.bfloat16(), table, lens, 2)),
        (TypeError, lambda: layer.attend_sparse(q, table, lens.long(), 2)),
        (ValueError, lambda: layer.attend_sparse(q, table, lens, 2, out=q.float())),
        (FkvLibraryError, lambda: layer.attend_sparse(q, table, lens, 2, scale=-1.0)),
        (FkvLibraryError, lambda: layer.attend_sparse(q, table, lens, 2, scale=float("inf"))),
        (ValueError, lambda: layer.bound(table, 0, -1)),
        (TypeError, lambda: layer.bound(table, torch.zeros(1, device="cuda"), 1)),
        (ValueError, lambda: layer.bound(table, torch.zeros(1, 2, dtype=torch.int32, device="cuda"), 2)),
        (TypeError, lambda: layer.bound(table.long(), 0, 1)),
        (ValueError, lambda: paged.PagedLayer.wrap("fp16", plain.k, plain.v, bounds=layer.bounds[:2])),
        (ValueError, lambda: paged.PagedLayer.wrap("fp16", plain.k, plain.v, bounds=layer.bounds.half())),
        (AttributeError, lambda: setattr(layer, "bounds", None)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("accepted", i)
    assert layer.attend_sparse(q[:0], table[:0], lens[:0], 2).shape == (0, 4, 1, 64)
    assert bool((layer.attend_sparse(q, table[:, :0], lens, 2) == 0).all())


def test_strides_and_streams(paged):
    layer = _with_bounds(paged, _filled(paged, "fp8", 40, 2, 64, 16, 80))
    table = _table(81, 40, [20, 20])
    layer.bound(table.cuda(), 0, 320)
    lens = [310, 77]
    q = _randn(82, 2, 6, 1, 64).half().cuda()
    want = _check(layer, q, table, lens, 6)
    for x in (torch.zeros(2, 6, 3, 64, dtype=torch.float16, device="cuda")[:, :, 1:2],
              torch.zeros(6, 2, 1, 64, dtype=torch.float16, device="cuda").transpose(0, 1),
              torch.zeros(2, 6, 1, 128, dtype=torch.float16, device="cuda")[..., ::2]):
        x.copy_(q)
        _bits_equal(layer.attend_sparse(x, table.cuda(), _i32(lens), 6), want, "strided query")
    x = q.clone()
    assert layer.attend_sparse(x, table.cuda(), _i32(lens), 6, out=x) is x
    _bits_equal(x, want, "in place")
    t, n = table.cuda(), _i32(lens)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        outs = [layer.attend_sparse(q, t, n, 6) for _ in range(10)]
    s.synchronize()
    for o in outs:
        _bits_equal(o, want, "side stream")


def test_captured_steps(paged):
    """A growing cache's steps, write with bounds and sparse attention, captured
    once for each of two caches and replayed side by side: the eager bits."""
    page, H, G, D, B, steps = 16, 2, 4, 128, 3, 40

    def cache(seed):
        layer = _with_bounds(paged, _filled(paged, "fp8", 60, H, D, page, seed))
        table = _table(seed + 1, 60, [20, 20, 20]).cuda()
        start = _i32([100, 7, 260])
        layer.bound(table, 0, 260, n_new=start)
        return layer, table, start, [tuple(_randn(seed + j + i, B, n, 1, D).bfloat16().cuda() for j, n in
                                           ((10, H), (100, H), (200, H * G))) for i in range(steps)]

    def step(layer, table, start, k, v, q):
        layer.write(k, v, table, start)
        return layer.attend_sparse(q, table, start, 5, lens_add=1, return_pages=True)

    eager = []
    for seed in (300, 700):
        layer, table, start, xs = cache(seed)
        eager.append([])
        for x in xs:
            eager[-1].append([t.clone() for t in step(layer, table, start, *x)])
            start.add_(1)
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
                start.add_(1)
        if i % 7 == 3:
            torch.cuda.synchronize()
            torch.randn(1000, device="cuda").sum().item()
        for (g, s, bufs, out, *_), want in zip(runs, eager):
            s.synchronize()
            for a, b in zip(out, want[i]):
                _bits_equal(a, b, f"replay {i}")
