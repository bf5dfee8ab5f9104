"""The paged KV cache on the GPU against 64-bit restatements: rotary
positions, writes and reads in every format bit for bit, one-token attention
within derived bounds; ragged lengths, empty sequences, pages outside the
pool, stale NaN rows, other streams, captured graphs."""

import math

import numpy as np
import pytest
import torch

import _paged_ref as ref

pytestmark = pytest.mark.gpu

FORMATS = ["fp16", "bf16", "fp8", "fp8_int4"]
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.load()
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def _flush(*a):
    print(*a, flush=True)


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def _table(seed, n_pages, counts, width=None):
    """Disjoint pages in random order; entries past a sequence's last are a
    page id that would be noticed."""
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(counts + [1]) if width is None else width
    t = torch.full((len(counts), width), 2 ** 31 - 1, dtype=torch.int32)
    for b, n in enumerate(counts):
        t[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return t


def _bits_equal(got, want, what):
    got, want = got.cpu(), want.cpu()
    same = (got == want) | (torch.isnan(got.float()) & torch.isnan(want.float()))
    assert bool(same.all()), f"{what}: {int((~same).sum())} of {same.numel()} differ"


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot,interleaved", [(64, 64, False), (128, 128, False), (128, 128, True), (64, 16, False),
                                               (128, 32, True), (80, 48, False), (512, 256, True), (16, 16, False)])
def test_rotary(paged, dtype, D, rot, interleaved):
    B, H, L = 3, 5, 7
    _flush("rotary", dtype, D, rot, interleaved)
    rope = paged.Rope(D, rot_dim=rot, interleaved=interleaved, max_positions=4096)
    x = _randn(1, B, L, H, D).to(dtype).cuda().transpose(1, 2)
    start = torch.tensor([0, 4000, 17], dtype=torch.int32)
    pos = start.numpy()[:, None] + np.arange(L)
    want = ref.rotate(ref.f64(x), pos, rope.table.cpu().numpy(), rot, interleaved)
    tol = (ref.UNIT[dtype] + 2.0 ** -24) * np.abs(want) * 1.001 + ref.TINY[dtype] + 2.0 ** -149
    for name, p in (("start", start.cuda()), ("start64", start.long().cuda()),
                    ("each", torch.from_numpy(pos).cuda()), ("each32", torch.from_numpy(pos).int().cuda())):
        got = rope(x, p)
        assert got.dtype == dtype and got.shape == x.shape
        assert (np.abs(ref.f64(got) - want) <= tol).all(), name
    # one start for all; in place, strided; a new tensor
    want = ref.rotate(ref.f64(x), np.broadcast_to(9 + np.arange(L), (B, L)), rope.table.cpu().numpy(), rot, interleaved)
    a = rope(x, 9)
    b = rope(x, torch.tensor(9, device="cuda"))
    c = x.clone()
    assert rope(c, 9, out=c) is c
    big = torch.full((B, H, L, D + 8), 7.0, dtype=dtype, device="cuda")
    d = big[..., :D]
    rope(x, 9, out=d)
    assert bool((big[..., D:] == 7).all())
    for got in (a, b, c, d):
        _bits_equal(got, a, "forms of one call")
    assert (np.abs(ref.f64(a) - want) <= (ref.UNIT[dtype] + 2.0 ** -24) * np.abs(want) * 1.001 + ref.TINY[dtype] + 2.0 ** -149).all()
    # unaligned rows (a view one element in) are copied first
    u = torch.empty(B * H * L * D + 1, dtype=dtype, device="cuda")[1:].view(B, H, L, D)
    u.copy_(x)
    _bits_equal(rope(u, 9), a, "unaligned input")
    o = torch.empty(B * H * L * D + 1, dtype=dtype, device="cuda")[1:].view(B, H, L, D)
    _bits_equal(rope(x, 9, out=o), a, "unaligned result")


@pytest.mark.parametrize("D,rot,scaling", [(128, 128, None), (64, 16, {"kind": "linear", "factor": 3.0}),
                                           (512, 512, {"kind": "yarn", "factor": 16.0, "original_positions": 4096})])
def test_rotary_table(paged, D, rot, scaling):
    """The device's table against the host's, far positions among it."""
    n = 70001
    rope = paged.Rope(D, rot_dim=rot, scaling=scaling, max_positions=n)
    inv, factor = paged._frequencies(rot, 10000.0, scaling)
    a = np.arange(n, dtype=np.float64)[:, None] * inv.numpy()
    t = ref.f64(rope.table)
    for got, want in ((t[:, 0], np.cos(a) * factor), (t[:, 1], np.sin(a) * factor)):
        # one rounding to fp32, and a sine of 64 bits
        assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want) * 1.001 + 2.0 ** -50).all()


def test_rotary_outside_the_table_and_empty(paged):
    rope = paged.Rope(64, rot_dim=32, max_positions=10)
    x = _randn(2, 1, 2, 4, 64).half().cuda()
    got = rope(x, torch.tensor([8], device="cuda"))
    assert bool(torch.isnan(got[:, :, 2:, :32]).all()) and not bool(torch.isnan(got[:, :, :2]).any())
    _bits_equal(got[..., 32:], x[..., 32:], "elements past rot_dim")
    assert bool(torch.isnan(rope(x, -1)[:, :, 0, :32]).all())
    assert rope(x[:, :, :0], 0).shape == (1, 2, 0, 64)
    assert rope(x[:0], torch.zeros(0, dtype=torch.int64, device="cuda")).shape == (0, 2, 4, 64)


# ---------------------------------------------------------------------------
# write and read
# ---------------------------------------------------------------------------

def _expected_pages(fmt, before, k, v, table, start, n_new, page, n_pages):
    """Page tensors (numpy) after a write of float64 rows that hold fp32
    numbers."""
    out = {n: t.cpu().clone() for n, t in before.items() if t is not None}
    B, H, L, D = k.shape
    for b in range(B):
        for i in range(int(n_new[b])):
            p = int(start[b]) + i
            if p < 0 or p >= table.shape[1] * page or not 0 <= int(table[b, p // page]) < n_pages:
                continue
            at = (int(table[b, p // page]), slice(None), p % page)
            if fmt in DTYPES:
                out["k"][at] = torch.from_numpy(k[b, :, i]).float().to(DTYPES[fmt])
                out["v"][at] = torch.from_numpy(v[b, :, i]).float().to(DTYPES[fmt])
                continue
            c, e = ref.e4m3_encode(k[b, :, i])
            out["k"][at], out["k_exp"][at] = torch.from_numpy(c), torch.from_numpy(e)
            if fmt == "fp8":
                c, e = ref.e4m3_encode(v[b, :, i])
                out["v"][at], out["v_scale"][at] = torch.from_numpy(c), torch.from_numpy(e)
            else:
                c, s, z = ref.int4_encode(v[b, :, i])
                out["v"][at] = torch.from_numpy(c[:, 0::2] | (c[:, 1::2] << 4))
                out["v_scale"][at] = torch.from_numpy(np.stack([s, z], -1))
    return out


def _tensors(layer):
    return {"k": layer.k, "v": layer.v, "k_exp": layer.k_exp, "v_scale": layer.v_scale}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,G,page,rot,interleaved", [(128, 4, 16, 128, False), (64, 7, 32, 32, True),
                                                      (128, 1, 64, 0, False)])
def test_write_and_read(paged, fmt, dtype, D, G, page, rot, interleaved):
    B, H, L = 4, 2, 9
    _flush("write", fmt, dtype, D, G, page, rot, interleaved)
    layer = paged.PagedLayer(13, H, D, page, fmt)
    for t in _tensors(layer).values():  # whatever was there stays
        if t is not None:
            t.copy_(torch.randint(1, 100, t.shape, generator=torch.Generator().manual_seed(3)).to(t.dtype))
    before = {n: None if t is None else t.clone() for n, t in _tensors(layer).items()}
    table = _table(4, 13, [3, 3, 3, 3])
    table[2, 1] = 13  # outside the pool
    table[3, 0] = -1
    start = torch.tensor([page - 4, 0, 2 * page - 3, 3 * page - 5])  # the last one runs past the table
    n_new = torch.tensor([9, 5, 9, 9])
    gain = torch.exp(2 * _randn(5, B, L, H, 1))
    k = (_randn(6, B, L, H, D) * gain).to(dtype).cuda().transpose(1, 2)
    v = (_randn(7, B, H, L, D) * 3 + 1).to(dtype).cuda()
    q = _randn(8, B, L, H * G, D).to(dtype).cuda().transpose(1, 2)
    rope = paged.Rope(D, rot_dim=rot, interleaved=interleaved, max_positions=4 * page) if rot else None
    qo = torch.full_like(q, 5.0)
    got_q = layer.write(k, v, table.cuda(), start.cuda(), n_new=n_new.int().cuda(), q=q, rope=rope, q_out=qo)
    assert got_q is qo
    pos = start.numpy()[:, None] + np.arange(L)
    k64, q64 = ref.f64(k), ref.f64(q)
    if rot:
        t = rope.table.cpu().numpy()
        k64, q64 = (ref.rotate(x, pos, t, rot, interleaved) for x in (k64, q64))
    want = _expected_pages(fmt, before, k64.astype(np.float32).astype(np.float64), ref.f64(v), table, start, n_new,
                           page, 13)
    for name, t in _tensors(layer).items():
        if t is not None:
            _bits_equal(t, want[name], name)
    past = (torch.arange(L) >= n_new[:, None])[:, None, :, None]
    want_q = torch.where(past, torch.tensor(5.0), torch.from_numpy(q64).float()).to(dtype)
    _bits_equal(qo, want_q, "q")
    # reads: the values that the pages stand for, rounded once
    lens = torch.tensor([page + 5, 1, 2 * page + 6, 0], dtype=torch.int32)
    values = ref.page_values(layer)
    for out_dtype, S in ((None, None), (torch.float32, 2 * page + 1), (torch.bfloat16, 3 * page + 10)):
        rk, rv = layer.read(table.cuda(), lens.cuda(), S, dtype=out_dtype)
        S = 3 * page if S is None else S
        assert rk.shape == rv.shape == (B, H, S, D)
        assert rk.dtype == (out_dtype or DTYPES.get(fmt, torch.float16))
        for b in range(B):
            n = min(int(lens[b]), S, 3 * page)
            rows, ok = ref.sequence(values, table.numpy(), b, n, page, 13)
            for got, w in zip((rk, rv), rows):
                w = np.where(ok[None, :, None], w, 0.0)
                g = ref.f64(got[b, :, :n])
                tol = (ref.UNIT[got.dtype] + 2.0 ** -24) * np.abs(w) + ref.TINY[got.dtype]
                # (an INT4 value is one fma in fp32)
                tol = tol + 2.0 ** -24 * np.abs(w)
                assert (np.abs(g - w) <= tol).all()
                assert bool((got[b, :, n:] == 0).all())


def test_every_e4m3_code_and_special_rows(paged):
    """Each code reads back as its value; rows of zeros, of one huge or tiny
    element, of infinities and NaN; -0; ties of the encoder."""
    layer = paged.PagedLayer(3, 1, 128, 16, "fp8")
    layer.k[0].copy_(torch.arange(2048).view(1, 16, 128) % 256)
    table = torch.tensor([[0]], dtype=torch.int32, device="cuda")
    k, _ = layer.read(table, torch.tensor([16], dtype=torch.int32, device="cuda"), dtype=torch.float32)
    _bits_equal(k[0, 0].view(-1), torch.from_numpy(ref.e4m3_value(np.arange(2048) % 256)).float(), "codes")
    rows = torch.zeros(16, 128, dtype=torch.float32)
    rows[1, 5] = 3.0e38
    rows[2, 5] = 1e-40
    rows[3] = _randn(9, 128)
    rows[3, 7] = math.inf
    rows[4] = _randn(10, 128)
    rows[4, 9] = math.nan
    rows[5] = -0.0
    rows[6, :] = 448.0
    rows[7, :] = 449.0
    rows[8, :17] = torch.tensor([(8 + m) * 2.0 ** -3 + 2.0 ** -4 for m in range(17)])  # ties
    rows[8, 100] = 448.0
    rows[9, :16] = torch.tensor([m * 2.0 ** -9 + 2.0 ** -10 for m in range(16)])  # subnormal ties
    rows[9, 100] = -300.0
    rows[10] = 224.0
    rows[11] = torch.nextafter(torch.tensor(224.0), torch.tensor(300.0))
    rows[12] = 2.0 ** -126
    rows[13] = _randn(11, 128) * 1e-37
    rows[14] = math.nan
    rows[15] = -math.inf
    x = rows.view(1, 1, 16, 128).cuda()
    for fmt in ("fp8", "fp8_int4"):
        layer = paged.PagedLayer(1, 1, 128, 16, fmt)
        layer.write(x, x, table, 0)
        c, e = ref.e4m3_encode(rows.double().numpy())
        got = layer.k[0, 0].cpu().numpy()
        assert np.array_equal(layer.k_exp[0, 0].cpu().numpy(), e)
        bad = ~np.isfinite(rows.numpy())
        assert (got[bad] & 127 == 127).all() and np.array_equal(got[~bad], c[~bad])
        k, v = layer.read(table, torch.tensor([16], dtype=torch.int32, device="cuda"), dtype=torch.float32)
        assert bool(torch.isnan(k[0, 0].cpu()[~torch.isfinite(rows)]).all())
        if fmt == "fp8_int4":
            plain = torch.isfinite(rows).all(-1)
            assert bool(torch.isnan(v[0, 0].cpu()[~plain]).all())
            cc, s, z = ref.int4_encode(rows[plain].double().numpy())
            packed = layer.v[0, 0].cpu().numpy()[plain.numpy()]
            assert np.array_equal(packed, cc[:, 0::2] | (cc[:, 1::2] << 4))
            assert np.array_equal(layer.v_scale[0, 0].cpu().numpy()[plain.numpy()], np.stack([s, z], -1))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _filled(paged, fmt, n_pages, H, D, page, seed, gain=1.0):
    """A layer whose every row is written, by the writer that the tests above
    hold to the codecs."""
    layer = paged.PagedLayer(n_pages, H, D, page, fmt)
    k, v = _randn(seed, n_pages, H, page, D), _randn(seed + 1, n_pages, H, page, D)
    k[..., 3] *= 6.0
    v = v * torch.exp(gain * _randn(seed + 2, n_pages, H, page, 1))
    ids = torch.arange(n_pages, dtype=torch.int32, device="cuda").view(n_pages, 1)
    layer.write(k.cuda(), v.cuda(), ids, 0)
    return layer


def _spoil(layer, table, lens):
    """NaN in every row that no sequence holds."""
    used = torch.zeros((layer.n_pages, layer.page_size), dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(max(n, 0)):
            i = int(table[b, p // layer.page_size]) if p // layer.page_size < table.shape[1] else -1
            if 0 <= i < layer.n_pages:
                used[i, p % layer.page_size] = True
    free = (~used).cuda()[:, None, :].expand(-1, layer.n_kv_heads, -1)
    nan8 = 127
    if layer.k_exp is None:
        layer.k[free] = math.nan
        layer.v[free] = math.nan
    else:
        layer.k[free] = nan8
        layer.k_exp[free] = 255
        layer.v[free] = nan8
        layer.v_scale[free] = 255 if layer.fmt == "fp8" else math.nan


def _check_attend(layer, q, table, lens, scale=None, **kw):
    out, lse = layer.attend(q, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=scale,
                            return_lse=True, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype
    s = layer.head_dim ** -0.5 if scale is None else scale
    add = kw.get("lens_add", 0)
    want, wlse, spread, ds = ref.attend(ref.f64(q)[:, :, 0], ref.page_values(layer), table.numpy(),
                                        [n + add for n in lens], layer.page_size, layer.n_pages, s)
    tol = ref.attend_bound(want, spread, ds, [n + add for n in lens], q.dtype)
    err = np.abs(ref.f64(out)[:, :, 0] - want)
    assert (err <= tol).all(), f"error {np.nanmax(err / tol)} of the bound, NaN {np.isnan(err).sum()}"
    g = ref.f64(lse)
    none = np.isinf(wlse)
    assert (g[none] == -np.inf).all()
    # lse: the score's error, the sum's, and its own rounding
    ltol = 2 * ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(np.where(none, 0.0, wlse))
    assert (np.abs(g[~none] - wlse[~none]) <= ltol[~none]).all()
    return out


EDGES = [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 255, 300]


@pytest.mark.parametrize("fmt,qd", [("fp16", "fp16"), ("bf16", "bf16"), ("fp8", "fp16"), ("fp8", "bf16"),
                                    ("fp8_int4", "fp16"), ("fp8_int4", "bf16")])
@pytest.mark.parametrize("D,H,G,page", [(128, 2, 4, 16), (64, 2, 7, 32), (128, 1, 1, 64), (64, 1, 16, 16),
                                        (128, 2, 20, 128), (64, 3, 33, 64)])
def test_attend_edges(paged, fmt, qd, D, H, G, page):
    _flush("attend", fmt, qd, D, H, G, page)
    counts = [-(-n // page) for n in EDGES]
    n_pages = sum(counts) + 2
    layer = _filled(paged, fmt, n_pages, H, D, page, 20)
    table = _table(21, n_pages, counts)
    _spoil(layer, table, EDGES)
    q = _randn(22, len(EDGES), 1, H * G, D).to(DTYPES[qd]).cuda().transpose(1, 2)
    out = _check_attend(layer, q, table, EDGES)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens", [[5003], [1, 9000, 3, 0, 2500], [777] * 40])
def test_attend_split(paged, fmt, lens):
    """Rows over several workgroups, each in its own way; sharp scores; the
    same bits whatever else runs, and with the bound given as max_len."""
    _flush("split", fmt, lens[:5])
    page, H, G, D = 32, 2, 5, 128
    counts = [-(-n // page) for n in lens]
    n_pages = sum(counts)
    layer = _filled(paged, fmt, n_pages, H, D, page, 30, gain=2.0)
    table = _table(31, n_pages, counts)
    q = (_randn(32, len(lens), H * G, 1, D) * 3).to(DTYPES.get(fmt, torch.bfloat16)).cuda()
    a = _check_attend(layer, q, table, lens)
    b = _check_attend(layer, q, table, lens, max_len=max(lens))
    c = _check_attend(layer, q, table, [n - 1 for n in lens], lens_add=1, max_len=max(lens))
    _check_attend(layer, q, table, lens, max_len=1)
    _check_attend(layer, q, table, lens, scale=-0.02)
    _bits_equal(b, c, "lens_add")
    for _ in range(3):
        _bits_equal(_check_attend(layer, q, table, lens), a, "again")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,H,G,B", [(128, 2, 4, 50), (64, 3, 5, 40), (64, 1, 40, 40)])
def test_attend_many_rows(paged, fmt, D, H, G, B):
    """Many rows of up to 1024 tokens, a workgroup each, and the same rows split
    (by a larger max_len), and longer ones than max_len says."""
    _flush("many rows", fmt, D, H, G, B)
    page, n = 64, [0, 1, 513, 1024, 130, 1023, 640, 900]
    lens = [n[b % len(n)] for b in range(B)]
    lens[3] = 1500
    counts = [-(-x // page) for x in lens]
    layer = _filled(paged, fmt, sum(counts) + 1, H, D, page, 38)
    table = _table(39, sum(counts) + 1, counts)
    _spoil(layer, table, lens)
    q = _randn(40, B, H * G, 1, D).to(DTYPES.get(fmt, torch.bfloat16)).cuda()
    for max_len in (1024, 513, 1500):
        out = _check_attend(layer, q, table, lens, max_len=max_len)
        assert bool((out[0] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,H,G", [(128, 1, 32), (128, 2, 17), (64, 1, 71)])
def test_attend_wide_groups(paged, fmt, D, H, G):
    """More than 16 heads on a KV head, over split rows: two tiles of heads a
    pass, the last one partly filled."""
    _flush("wide", fmt, D, H, G)
    lens, page = [700, 1, 0, 3001], 64
    counts = [-(-n // page) for n in lens]
    layer = _filled(paged, fmt, sum(counts) + 1, H, D, page, 35)
    table = _table(36, sum(counts) + 1, counts)
    _spoil(layer, table, lens)
    q = _randn(37, 4, H * G, 1, D).to(DTYPES.get(fmt, torch.float16)).cuda()
    out = _check_attend(layer, q, table, lens)
    assert bool((out[2] == 0).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_attend_pages_outside_the_pool_and_long_lens(paged, fmt):
    page, H, G, D = 16, 2, 3, 64
    layer = _filled(paged, fmt, 30, H, D, page, 40)
    table = _table(41, 30, [10, 10, 10])
    table[0, 3], table[0, 9], table[1, 0], table[2, :] = -1, 30, 2 ** 30, -7
    lens = [160, 10 ** 6, 100]  # the second one is longer than its table
    q = _randn(42, 3, H * G, 1, D).to(DTYPES.get(fmt, torch.float16)).cuda()
    out = _check_attend(layer, q, table, lens)
    assert bool((out[2] == 0).all())
    _check_attend(layer, q, table, [-3, -2 ** 31, 0])


def test_attend_nan_of_one_sequence_stays_there(paged):
    layer = _filled(paged, "bf16", 20, 1, 128, 16, 50)
    table = _table(51, 20, [10, 10])
    layer.v[int(table[0, 4]), 0, 3, 77] = math.nan
    layer.k[int(table[0, 9]), 0, 0, 0] = math.inf
    q = _randn(52, 2, 8, 1, 128).bfloat16().cuda()
    lens = torch.tensor([145, 145], dtype=torch.int32, device="cuda")
    out = layer.attend(q, table.cuda(), lens)
    # an infinite key scores +inf (all NaN) or, where the query is negative,
    # -inf: it takes no part, and the NaN value is one dim's
    nan = torch.isnan(out).cpu()
    up = q[0, :, 0, 0].cpu() > 0
    assert 0 < int(up.sum()) < 8
    assert bool(nan[0, up].all()) and nan[0, ~up].nonzero()[:, -1].unique().tolist() == [77]
    assert not bool(nan[1].any())
    lens[0] = 64  # before both
    assert not bool(torch.isnan(layer.attend(q, table.cuda(), lens)).any())


def test_attend_scores_at_the_edge_of_fp32(paged):
    """Scores near -3e38 and far apart: a softmax like any other (a maximum
    that starts above them would leave no weight)."""
    H, D, page = 1, 64, 16
    layer = paged.PagedLayer(40, H, D, page, "bf16")
    layer.k.fill_(0.0)
    layer.k[..., 0] = -1.0e18
    layer.k[1, 0, 3, 0] = -0.5e18
    layer.v.copy_(_randn(65, 40, H, page, D))
    table = torch.arange(40, dtype=torch.int32).view(1, 40)
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16, device="cuda")
    q[0, :, 0, 0] = 1.0e18
    for n in (10, 640):  # whole, split
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        out, lse = layer.attend(q, table.cuda(), lens, scale=128.0, return_lse=True)
        v = layer.v.float().cpu().transpose(1, 2).reshape(-1, D)[:n]
        want = v.double().mean(0) if n < 20 else layer.v[1, 0, 3].double().cpu()
        err = (out[0, :, 0].double().cpu() - want).abs()
        # equal weights or a single one: exact but for fp32 sums and the result's rounding
        assert bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * v.abs().max()).all())
        # -128 * 1e18 * 1e18 (the bf16 numbers) or half of it
        s = 128.0 * float(q[0, 0, 0, 0]) * float(layer.k[0, 0, 0, 0] if n < 20 else layer.k[1, 0, 3, 0])
        assert bool(((lse.cpu().double() - s).abs() <= 2.0 ** -20 * abs(s)).all())


def test_attend_many_sequences(paged):
    """More sequences than a workgroup has threads, most of them empty."""
    B, page, H, D = 700, 16, 2, 64
    lens = [0] * B
    for i, n in ((3, 40), (255, 1), (256, 17), (257, 300), (699, 130)):
        lens[i] = n
    counts = [-(-n // page) for n in lens]
    layer = _filled(paged, "fp16", sum(counts), H, D, page, 60)
    table = _table(61, sum(counts), counts)
    _check_attend(layer, _randn(62, B, H * 2, 1, D).half().cuda(), table, lens)


def test_attend_shared_pages_and_queries(paged):
    """A prefix that two sequences share, and one query broadcast to all."""
    layer = _filled(paged, "fp8", 12, 2, 128, 16, 70)
    table = _table(71, 12, [6, 6])
    table[1, :4] = table[0, :4]
    q = _randn(72, 1, 8, 1, 128).half().cuda().expand(2, -1, -1, -1)
    _check_attend(layer, q, table, [90, 70])
    lens = torch.tensor([60, 60], dtype=torch.int32, device="cuda")
    out = layer.attend(q, table.cuda(), lens)
    _bits_equal(out[0], out[1], "equal prefixes")


def test_far_offsets(paged):
    """Pages that lie past 2^31 bytes and elements of the pool."""
    page, H, D = 64, 8, 128
    n_pages = 36000  # 2.4e9 codes
    layer = paged.PagedLayer(n_pages, H, D, page, "fp8")
    ids = [n_pages - 1, 0, n_pages - 2]
    table = torch.tensor([ids], dtype=torch.int32)
    k, v = (_randn(80 + i, 1, H, 3 * page, D).bfloat16().cuda() for i in range(2))
    layer.write(k, v, table.cuda(), 0)
    lens = torch.tensor([3 * page - 1], dtype=torch.int32, device="cuda")
    rk, rv = layer.read(table.cuda(), lens, dtype=torch.float32)
    small = paged.PagedLayer(3, H, D, page, "fp8")
    t3 = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    small.write(k, v, t3.cuda(), 0)
    q = _randn(82, 1, 32, 1, D).bfloat16().cuda()
    for got, want in zip((rk, rv, layer.attend(q, table.cuda(), lens)),
                         (*small.read(t3.cuda(), lens, dtype=torch.float32), small.attend(q, t3.cuda(), lens))):
        _bits_equal(got, want, "far pages")


# ---------------------------------------------------------------------------
# streams, graphs
# ---------------------------------------------------------------------------

def _step(layer, rope, k, v, q, table, start):
    qr = layer.write(k, v, table, start, q=q, rope=rope)
    return layer.attend(qr, table, start, lens_add=1)


@pytest.mark.parametrize("fmt", ["bf16", "fp8_int4"])
def test_steps_captured_on_two_streams(paged, fmt):
    """Decode steps of two caches, each captured once, replayed side by side
    on two streams while both caches grow: the eager result's bits."""
    _flush("graphs", fmt)
    page, H, G, D, B, steps = 16, 2, 4, 128, 3, 40
    rope = paged.Rope(D, max_positions=4096)

    def cache(seed):
        layer = _filled(paged, fmt, 20 * B, H, D, page, seed)
        table = _table(seed + 1, 20 * B, [20] * B).cuda()
        xs = [(_randn(seed + 10 + i, B, H, 1, D).bfloat16().cuda(), _randn(seed + 100 + i, B, H, 1, D).bfloat16().cuda(),
               _randn(seed + 200 + i, B, H * G, 1, D).bfloat16().cuda()) for i in range(steps)]
        return layer, table, torch.tensor([100, 7, 260], dtype=torch.int32, device="cuda"), xs

    eager = []
    for seed in (300, 700):
        layer, table, start, xs = cache(seed)
        eager.append([])
        for x in xs:
            eager[-1].append(_step(layer, rope, *x, table, start).clone())
            start.add_(1)
    torch.cuda.synchronize()
    runs = []
    for seed in (300, 700):
        layer, table, start, xs = cache(seed)
        bufs = [t.clone() for t in xs[0]]
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            out = _step(layer, rope, *bufs, table, start)
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
            _bits_equal(out, want[i], f"replay {i}")


def test_another_stream_than_the_current_one(paged):
    layer = _filled(paged, "fp8", 10, 2, 64, 16, 90)
    table = _table(91, 10, [5, 5]).cuda()
    lens = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    q = _randn(92, 2, 6, 1, 64).half().cuda()
    want = layer.attend(q, table, lens)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        outs = [layer.attend(q, table, lens) for _ in range(10)]
    s.synchronize()
    for o in outs:
        _bits_equal(o, want, "side stream")
