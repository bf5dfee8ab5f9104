"""The paged cache without a GPU: rotary frequencies against their formulas,
the page table's bookkeeping, and every refusal of the C entry points and of
the Python ones that takes no device."""

import ctypes
import math

import pytest
import torch

import _paged_ref as ref
from foveated_kv_amd import PagedKVCache, PageTable, Rope, _lib, paged


# ---------------------------------------------------------------------------
# rotary tables
# ---------------------------------------------------------------------------

def _angle_rates(rot, base, scaling):
    out = []
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        kind = scaling and scaling["kind"]
        if kind == "linear":
            f /= scaling["factor"]
        elif kind == "ntk":
            f = (base * scaling["factor"] ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif kind == "bands":
            turns = scaling["original_positions"] * f / (2 * math.pi)
            lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
            if turns < lo:
                f /= scaling["factor"]
            elif turns < hi:
                t = (turns - lo) / (hi - lo)
                f = t * f + (1 - t) * f / scaling["factor"]
        elif kind == "yarn":
            def at(beta):
                return rot * math.log(scaling["original_positions"] / (beta * 2 * math.pi)) / (2 * math.log(base))
            lo = max(math.floor(at(scaling["beta_fast"])), 0)
            hi = min(math.ceil(at(scaling["beta_slow"])), rot // 2 - 1)
            t = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
            f = t * f / scaling["factor"] + (1 - t) * f
        out.append(f)
    return out, (0.1 * math.log(scaling["factor"]) + 1) if scaling and scaling["kind"] == "yarn" else 1.0


SCALINGS = [None, {"kind": "linear", "factor": 4.0}, {"kind": "ntk", "factor": 8.0},
            {"kind": "bands", "factor": 8.0, "original_positions": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0},
            {"kind": "yarn", "factor": 16.0, "original_positions": 4096, "beta_fast": 32.0, "beta_slow": 1.0}]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("rot,base", [(128, 10000.0), (64, 500000.0), (16, 10000.0)])
def test_rope_table(scaling, rot, base):
    rope = Rope(128, rot_dim=rot, base=base, scaling=scaling, max_positions=70000, device="cpu")
    assert rope.table.shape == (70000, 2, rot // 2) and rope.table.dtype == torch.float32
    rates, factor = _angle_rates(rot, base, scaling)
    for p in (0, 1, 77, 4095, 65535, 65536, 69999):
        for i, f in enumerate(rates):
            # one rounding to fp32, and an angle of 64 bits: p f is off by a few 2^-53 of it
            tol = 2.0 ** -24 * factor * 1.001 + 8 * 2.0 ** -53 * p
            assert abs(float(rope.table[p, 0, i]) - factor * math.cos(p * f)) <= tol
            assert abs(float(rope.table[p, 1, i]) - factor * math.sin(p * f)) <= tol


@pytest.mark.parametrize("kw", [{"rot_dim": 8}, {"rot_dim": 40}, {"rot_dim": 144}, {"base": 1.0}, {"base": math.inf},
                                {"max_positions": 0}, {"scaling": {"kind": "nope", "factor": 2.0}},
                                {"scaling": {"kind": "linear", "factor": 0.5}}, {"scaling": {"kind": "linear"}},
                                {"scaling": {"kind": "linear", "factor": 2.0, "beta_fast": 1.0}},
                                {"scaling": {"kind": "yarn", "factor": 2.0}},
                                {"scaling": {"kind": "bands", "factor": 2.0, "original_positions": 10,
                                             "low_freq_factor": 4.0, "high_freq_factor": 4.0}}])
def test_rope_refusals(kw):
    with pytest.raises(ValueError):
        Rope(128, device="cpu", **kw)


def test_cpu_tensors_are_refused():
    rope = Rope(64, max_positions=8, device="cpu")
    with pytest.raises(TypeError, match="ROCm device"):
        rope(torch.zeros(1, 1, 1, 64))
    with pytest.raises(TypeError, match="ROCm device"):
        paged.PagedLayer(2, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="fmt"):
        paged.PagedLayer(2, 1, 64, fmt="int3", device="cpu")
    with pytest.raises(ValueError, match="head dim"):
        PagedKVCache(1, 1, 128, 4, rope=rope, device="cpu")


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------

def _state(t):
    return [t.pages(b) for b in range(t.max_seqs)], t.lengths(), t.starts(), t.free_pages, t.table.clone()


def _check(t):
    held = [p for b in range(t.max_seqs) for p in t.pages(b)]
    assert len(held) == len(set(held)) and sorted(held + t._free) == list(range(t.n_pages))
    for b in range(t.max_seqs):
        row = t.table[b].tolist()
        n = len(t.pages(b))
        assert row[:n] == t.pages(b) and all(x == -1 for x in row[n:])
        assert t.lens[b] == t.lengths()[b] <= n * t.page_size
        assert t.start[b] == t.starts()[b] and t.new[b] == t.lens[b] - t.start[b]


def test_page_table_grows_and_frees():
    t = PageTable(12, 16, 3, 100, device="cpu")
    assert t.table.shape == (3, 7)
    t.extend([5, 16, 0])
    _check(t)
    assert t.lengths() == [5, 16, 0] and [len(t.pages(b)) for b in range(3)] == [1, 1, 0]
    for _ in range(12):
        t.extend(1)
        _check(t)
    assert t.lengths() == [17, 28, 12] and t.starts() == [16, 27, 11]
    t.extend(20, slice(1, 2))
    _check(t)
    t.reserve(80, slice(2, 3))
    assert len(t.pages(2)) == 5 and t.lengths()[2] == 12
    _check(t)
    before = _state(t)
    for bad in (lambda: t.extend(60), lambda: t.extend([0, 0, 89]), lambda: t.reserve(101, slice(0, 1))):
        with pytest.raises(MemoryError):
            bad()
        after = _state(t)
        assert after[:4] == before[:4] and torch.equal(after[4], before[4])
    t.free(1)
    t.free(1)
    _check(t)
    assert t.lengths() == [17, 0, 12]
    t.extend([1, 48, 1])
    _check(t)
    for bad in (lambda: t.extend(-1), lambda: t.extend([1, 2]), lambda: t.free(3), lambda: t.extend(1, slice(0, 3, 2)),
                lambda: t.reserve([1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError):
        PageTable(0, 16, 1, 10, device="cpu")


# ---------------------------------------------------------------------------
# C entry points
# ---------------------------------------------------------------------------

@pytest.fixture()
def c():
    """Arguments that would pass, over memory that no refused call touches."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(8192)
    at = (ctypes.addressof(buf) + 255) & ~255

    class C:
        pass

    o = C()
    o.lib, o.buf, o.at = lib, buf, at
    o.pages = lambda **kw: _lib.PagesC(**{**dict(k=at, v=at, k_exp=at, v_scale=at, n_pages=2, page_size=16, H=2, D=64,
                                                 format=2), **kw})
    o.rows = lambda **kw: _lib.RowsC(**{**dict(data=at, stride_b=128, stride_h=64, stride_l=64), **kw})
    o.pos = lambda **kw: _lib.PositionsC(**{**dict(data=None), **kw})
    o.rope = lambda **kw: _lib.RopeC(**{**dict(table=at, n_positions=4, rot_dim=32, interleaved=0), **kw})
    return o


def _refused(rc, lib, word):
    assert rc == _lib.FKV_EINVAL and word in lib.fkv_last_error().decode(), lib.fkv_last_error()


R = ctypes.byref


@pytest.mark.parametrize("word,kw", [
    ("NULL rope", {"rope": None}), ("dtype", {"dtype": 3}), ("negative", {"B": -1}), ("negative", {"L": -5}),
    ("head dim", {"D": 8}), ("head dim", {"D": 100}), ("head dim", {"D": 520}), ("rot_dim", {"rope": {"rot_dim": 24}}),
    ("rot_dim", {"rope": {"rot_dim": 80}}), ("rot_dim", {"rope": {"rot_dim": 0}}), ("table", {"rope": {"table": None}}),
    ("no positions", {"rope": {"n_positions": 0}}), ("NULL positions", {"pos": None}),
    ("misaligned", {"pos": {"data": 0x1002}}), ("misaligned", {"pos": {"data": 0x1004, "is64": 1}}),
    ("2^31", {"B": 65536, "L": 65536}), ("too many", {"H": 1, "L": 1 << 27}), ("NULL rows", {"x": None}),
    ("NULL rows", {"out": {"data": None}}), ("aligned", {"x": {"data": 0x1008}}), ("multiples", {"out": {"stride_l": 60}})])
def test_rope_apply_refusals(c, word, kw):
    a = dict(rope={}, x={}, out={}, pos={}, dtype=0, B=1, H=2, L=3, D=64, **{})
    a.update(kw)
    args = {n: None if a[n] is None else R(getattr(c, "rows" if n in ("x", "out") else n)(**a[n]))
            for n in ("rope", "x", "out", "pos")}
    rc = c.lib.fkv_rope_apply(args["rope"], args["x"], args["out"], a["dtype"], a["B"], a["H"], a["L"], a["D"],
                              args["pos"], None)
    _refused(rc, c.lib, word)


@pytest.mark.parametrize("word,kw", [("NULL", {"f": None}), ("NULL", {"table": None}), ("misaligned", {"table": 0x1004}),
                                     ("rot_dim", {"rot": 24}), ("rot_dim", {"rot": 528}), ("no positions", {"n": 0})])
def test_rope_table_refusals(c, word, kw):
    a = {"f": c.at, "rot": 32, "n": 4, "table": c.at, **kw}
    _refused(c.lib.fkv_rope_table(a["f"], a["rot"], 1.0, a["n"], a["table"], None), c.lib, word)


BAD_PAGES = [("head dim", {"D": 96}), ("format", {"format": 4}), ("format", {"format": -1}), ("power of two", {"page_size": 8}),
             ("power of two", {"page_size": 48}), ("power of two", {"page_size": 2048}), ("count", {"n_pages": 0}),
             ("count", {"H": 0}), ("count", {"H": 1025}), ("NULL", {"k": None}), ("NULL", {"v": None}),
             ("NULL", {"k_exp": None}), ("NULL", {"v_scale": None}), ("aligned", {"k": 0x1008}), ("aligned", {"v_scale": 0x1004})]


@pytest.mark.parametrize("word,kw", BAD_PAGES)
def test_page_refusals(c, word, kw):
    pg, r, p = c.pages(**kw), c.rows(), c.pos()
    _refused(c.lib.fkv_paged_write(R(pg), R(r), R(r), 0, 1, 1, c.at, 1, 1, R(p), None, None, None, None, 0, None),
             c.lib, word)
    _refused(c.lib.fkv_paged_read(R(pg), c.at, 1, 1, c.at, 1, 1, c.at, c.at, 0, None), c.lib, word)
    _refused(c.lib.fkv_paged_attn_workspace(R(pg), 2, 1, 16), c.lib, word)
    _refused(c.lib.fkv_paged_attn(R(pg), R(r), 0, 2, 1, c.at, 1, 1, c.at, 0, 16, 1.0, c.at, None, c.at, 1 << 30, None),
             c.lib, word)
    _refused(c.lib.fkv_paged_attn_workspace(None, 2, 1, 16), c.lib, "NULL pages")


@pytest.mark.parametrize("word,kw", [
    ("dtype", {"dtype": 5}), ("negative", {"L": -1}), ("table shape", {"B": -1}), ("table shape", {"n_table": -1}),
    ("table shape", {"B": 2, "n_table": 4, "stride": 3}), ("NULL table", {"table": None}), ("NULL positions", {"pos": None}),
    ("one position", {"pos": {"per_token": 1}}), ("together", {"q": {}}), ("together", {"q_out": {}}),
    ("query head", {"q": {}, "q_out": {}, "Hq": 0}), ("rot_dim", {"rope": {"rot_dim": 72}}), ("NULL rows", {"k": None}),
    ("aligned", {"v": {"data": 0x1001}}), ("multiples", {"k": {"stride_h": 63}}), ("2^31", {"B": 40000, "L": 40000}),
    ("too many", {"B": 1 << 14, "L": 18000}), ("aligned", {"q": {"data": 0x1008}, "q_out": {}, "Hq": 2})])
def test_write_refusals(c, word, kw):
    a = dict(k={}, v={}, q=None, q_out=None, pos={}, rope=None, dtype=0, B=1, L=1, table=c.at, n_table=1, stride=1, Hq=0)
    a.update(kw)
    s = {n: None if a[n] is None else R(getattr(c, {"pos": "pos", "rope": "rope"}.get(n, "rows"))(**a[n]))
         for n in ("k", "v", "q", "q_out", "pos", "rope")}
    rc = c.lib.fkv_paged_write(R(c.pages()), s["k"], s["v"], a["dtype"], a["B"], a["L"], a["table"], a["n_table"],
                               a["stride"], s["pos"], None, s["rope"], s["q"], s["q_out"], a["Hq"], None)
    _refused(rc, c.lib, word)


@pytest.mark.parametrize("word,kw", [
    ("dtype", {"dtype": -1}), ("negative", {"S": -1}), ("table shape", {"stride": 0, "B": 2}), ("NULL table", {"table": None}),
    ("lens", {"lens": None}), ("aligned", {"k": None}), ("aligned", {"v": 0x1008}), ("2^31", {"S": 2 ** 31 - 1}),
    ("too many", {"B": 300_000_000, "stride": 1, "S": 2})])
def test_read_refusals(c, word, kw):
    a = dict(table=c.at, n_table=1, stride=1, lens=c.at, B=1, S=1, k=c.at, v=c.at, dtype=0)
    a.update(kw)
    rc = c.lib.fkv_paged_read(R(c.pages()), a["table"], a["n_table"], a["stride"], a["lens"], a["B"], a["S"], a["k"],
                              a["v"], a["dtype"], None)
    _refused(rc, c.lib, word)


@pytest.mark.parametrize("word,kw", [
    ("sequences", {"B": 4097}), ("sequences", {"B": -1}), ("multiple", {"Hq": 3}), ("multiple", {"Hq": 0}),
    ("max_len", {"max_len": -1}), ("table shape", {"n_table": -1}), ("2^31 tokens", {"n_table": 2 ** 27}), ("2^24 rows", {"B": 4096, "Hq": 2 ** 18, "max_len": 100}),
    ("2^31 tiles", {"B": 4096, "Hq": 2 ** 14, "n_table": 2 ** 20, "max_len": 100}),
    ("fp16 or bf16", {"q_dtype": 2}), ("16-bit pages' type", {"format": 0, "q_dtype": 1}),
    ("16-bit pages' type", {"format": 1, "q_dtype": 0}), ("finite", {"scale": math.nan}), ("finite", {"scale": math.inf}),
    ("NULL", {"q": None}), ("NULL", {"out": None}), ("NULL", {"lens": None}), ("aligned", {"q": {"data": 0x1008}}),
    ("aligned", {"out": 0x1008}), ("multiples", {"q": {"stride_h": 60}}), ("workspace", {"ws": None}),
    ("workspace", {"ws_bytes": 16}), ("NULL table", {"table": None})])
def test_attn_refusals(c, word, kw):
    a = dict(format=2, q={}, q_dtype=0, Hq=4, B=1, table=c.at, n_table=64, stride=2 ** 27, lens=c.at, max_len=65536,
             scale=1.0, out=c.at, ws=c.at, ws_bytes=1 << 40)
    a.update(kw)
    rc = c.lib.fkv_paged_attn(R(c.pages(format=a["format"])), None if a["q"] is None else R(c.rows(**a["q"])),
                              a["q_dtype"], a["Hq"], a["B"], a["table"], a["n_table"], a["stride"], a["lens"], 0,
                              a["max_len"], a["scale"], a["out"], None, a["ws"], a["ws_bytes"], None)
    _refused(rc, c.lib, word)


def test_empty_calls_do_nothing(c):
    """No rows: accepted without a launch (there is no device here)."""
    pg, r, p, rope = c.pages(), c.rows(), c.pos(), c.rope()
    assert c.lib.fkv_rope_apply(R(rope), None, None, 0, 0, 2, 3, 64, R(p), None) == 0
    assert c.lib.fkv_paged_write(R(pg), None, None, 0, 0, 1, None, 1, 1, R(p), None, None, None, None, 0, None) == 0
    assert c.lib.fkv_paged_write(R(pg), None, None, 0, 1, 0, c.at, 1, 1, R(p), None, None, None, None, 0, None) == 0
    assert c.lib.fkv_paged_read(R(pg), c.at, 1, 1, None, 1, 0, None, None, 0, None) == 0
    assert c.lib.fkv_paged_attn(R(pg), None, 0, 4, 0, None, 1, 1, None, 0, 0, 1.0, None, None, None, 0, None) == 0


def test_workspace_covers_every_length(c):
    """No bound on the lengths asks for more than the largest, and no device
    is needed to know."""
    for H, Hq, D in ((2, 4, 64), (8, 64, 128), (1, 40, 128)):
        pg = c.pages(H=H, D=D)
        for B in (1, 7, 64):
            sizes = [c.lib.fkv_paged_attn_workspace(R(pg), Hq, B, n) for n in (0, 1, 128, 129, 4096, 2 ** 20)]
            assert all(0 <= s <= 1 << 27 for s in sizes)


def test_reference_codecs():
    """The oracle's own codec against the definition: every level is nearest."""
    import numpy as np

    rows = np.random.default_rng(0).normal(size=(50, 64)).astype(np.float32).astype(np.float64) * 10
    codes, exps = ref.e4m3_encode(rows)
    e = exps.astype(np.int64) - 127
    u = rows * 2.0 ** -e[:, None]
    assert ((np.abs(u).max(-1) <= 448) & (np.abs(u).max(-1) > 224)).all()
    got = ref.e4m3_value(codes)
    every = ref.e4m3_value(np.array([c for c in range(256) if c & 127 != 127]))
    best = np.abs(u[..., None] - every).min(-1)
    assert np.array_equal(np.abs(u - got), best)
    t = torch.from_numpy(u).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(t, codes)
    c, s, z = ref.int4_encode(rows)
    back = c * s[:, None].astype(np.float64) + z[:, None]
    # half a step, and the scale's rounding 15 times over
    assert (np.abs(back - rows) <= s[:, None] * (0.5 + 15 * 2.0 ** -24) * 1.0000001).all()


# ---------------------------------------------------------------------------
# results and model calls
# ---------------------------------------------------------------------------

def test_results_whose_rows_share_memory_are_refused():
    x = torch.zeros(2, 3, 5, 64)
    shape, dtype = x.shape, x.dtype
    paged._result(-1, "out", x, shape, dtype)
    paged._result(-1, "out", torch.zeros(2, 5, 3, 64).transpose(1, 2), shape, dtype)
    one = torch.zeros(1, 3, 5, 64)
    # (one sequence: its stride says nothing)
    paged._result(-1, "out", one.as_strided(one.shape, (0, 320, 64, 1)), one.shape, dtype)
    for bad in (x[:1].expand(2, -1, -1, -1), x[:, :1].expand(-1, 3, -1, -1), x[..., :1].expand(-1, -1, -1, 64), x[:1],
                x.half()):
        with pytest.raises(ValueError):
            paged._result(-1, "out", bad, shape, dtype)


def test_attention_call_must_have_the_written_tokens():
    from foveated_kv_amd import generate

    class Cache:
        rope, layers, pages = None, [None], PageTable(4, 16, 2, 32, device="cpu")
        written = 0

        def write(self, *args, **kw):
            Cache.written += 1

    cache = Cache()
    kv, original = torch.zeros(2, 1, 5, 64), torch.nn.functional.scaled_dot_product_attention
    w, = generate.install_paged_attention(cache)
    try:
        for keys, queries in ((kv[:, :, :1], kv), (kv, kv[:, :, :1]), (kv, kv[:, :, :4]), (kv[:, :, :1], kv[0])):
            w.update_and_fetch(keys, keys)
            with pytest.raises(RuntimeError, match="update_and_fetch took"):
                torch.nn.functional.scaled_dot_product_attention(queries, keys, keys)
        assert Cache.written == 2
        k, v = w.update_and_fetch(kv, kv)
        torch.nn.functional.scaled_dot_product_attention(kv, k, v)
        torch.nn.functional.scaled_dot_product_attention(kv[0], kv[0], kv[0])  # (another attention than the cache's)
    finally:
        generate.uninstall_paged_attention()
    assert torch.nn.functional.scaled_dot_product_attention is original


def test_compiled_calls_leave_what_is_not_plain():
    calls, x = _lib.calls(), torch.zeros(2, 3, 5, 64)
    rope = Rope(64, max_positions=8, device="cpu")
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: calls.rope(rope._key, x, 0, None), lambda: calls.rope(rope._key, None, "0", 3), lambda: calls.rope(),
                 lambda: calls.rope(None, x, 0, None), lambda: calls.rope((1, 2), x, 2 ** 70, None),
                 lambda: calls.write((0, 0), x, x, i[None], 0, None, None, None, None), lambda: calls.write((0, 0)),
                 lambda: calls.read((0, 0), i[None], i, None, None), lambda: calls.read("pages", 1, 2, 3, 4),
                 lambda: calls.attend((0, 0), x, i[None], i, None, 0, None, None, False), lambda: calls.attend(*[x] * 9)):
        assert call() is NotImplemented


def test_compiled_calls_that_are_missing_raise(monkeypatch):
    import sys

    import foveated_kv_amd

    monkeypatch.setattr(_lib, "_calls", None)
    monkeypatch.setitem(sys.modules, "foveated_kv_amd._fkv_calls", None)
    monkeypatch.delattr(foveated_kv_amd, "_fkv_calls", raising=False)
    with pytest.raises(_lib.FkvLibraryError, match="make -C"):
        _lib.calls()
