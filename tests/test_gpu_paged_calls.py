"""The paged cache's compiled calls against the ones in Python: the same bits
for every form of argument that they take, and nothing done for one that they
leave."""

import pytest
import torch

pytestmark = pytest.mark.gpu

B, H, G, L, D, PAGE = 3, 2, 4, 5, 64, 16


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.calls()
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


class _Left:
    """Leaves every call to Python."""

    def __getattr__(self, name):
        return lambda *args: NotImplemented


class _Counting:
    def __init__(self, calls):
        self.calls, self.done = calls, []

    def __getattr__(self, name):
        def call(*args):
            r = getattr(self.calls, name)(*args)
            self.done.append(r is not NotImplemented)
            return r
        return call


def _both(monkeypatch, run, plain):
    """run() by way of the compiled calls and without them -> both results."""
    from foveated_kv_amd import _lib

    seen = _Counting(_lib.calls())
    monkeypatch.setattr(_lib, "calls", lambda: seen)
    got = run()
    assert seen.done == [plain], f"compiled calls done {seen.done}, expected {[plain]}"
    monkeypatch.setattr(_lib, "calls", _Left)
    want = run()
    monkeypatch.undo()
    flat = [r if isinstance(r, (tuple, list)) else [r] for r in (got, want)]
    assert len(flat[0]) == len(flat[1])
    for a, b in zip(*flat):
        if a is None or b is None:
            assert a is b
            continue
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and a.device == b.device
        assert torch.equal(torch.nan_to_num(a.float(), 1e9), torch.nan_to_num(b.float(), 1e9))
    return got


def _randn(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to("cuda", dtype)


def _i(*v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


POSITIONS = {
    "number": (True, lambda: 7),
    "true": (True, lambda: True),
    "scalar": (True, lambda: _i(3, dtype=torch.int64)[0]),
    "one": (True, lambda: _i(3)),
    "each": (True, lambda: _i(0, 9, 20)),
    "each64": (True, lambda: _i(0, 9, 20, dtype=torch.int64)),
    "strided": (True, lambda: _i(0, 1, 9, 1, 20, 1)[::2]),
    "outside": (True, lambda: _i(-5, 60, 2 ** 31 - 1)),
    "token": (True, lambda: torch.arange(B * L, device="cuda").view(B, L)),
    "row": (True, lambda: torch.arange(L, device="cuda", dtype=torch.int32)[None]),
    "numpy": (False, lambda: __import__("numpy").int64(4)),
}


@pytest.mark.parametrize("name", POSITIONS)
def test_rotary_positions(paged, monkeypatch, name):
    plain, make = POSITIONS[name]
    rope, x, pos = paged.Rope(D, max_positions=64), _randn(1, B, H, L, D), make()
    _both(monkeypatch, lambda: rope(x, pos), plain)


ROWS = {
    "contiguous": (True, lambda dt: _randn(2, B, H, L, D, dtype=dt)),
    "tokens first": (True, lambda dt: _randn(2, B, L, H, D, dtype=dt).transpose(1, 2)),
    "part": (True, lambda dt: _randn(2, B, H, L + 3, D + 64, dtype=dt)[:, :, 1:L + 1, 64:]),
    "expanded": (True, lambda dt: _randn(2, B, 1, L, D, dtype=dt).expand(-1, H, -1, -1)),
    "unaligned": (False, lambda dt: _randn(2, B, H, L, D + 8, dtype=dt)[..., 1:D + 1]),
    "dims strided": (False, lambda dt: _randn(2, B, H, D, L, dtype=dt).transpose(2, 3)),
    "empty": (True, lambda dt: _randn(2, 0, H, L, D, dtype=dt)),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ROWS)
def test_rotary_rows(paged, monkeypatch, name, dtype):
    plain, make = ROWS[name]
    rope, x = paged.Rope(D, rot_dim=32, interleaved=True, max_positions=64), make(dtype)
    n = x.shape[0]
    _both(monkeypatch, lambda: rope(x, 5), plain)
    out = torch.zeros(n, L, H, D, dtype=dtype, device="cuda").transpose(1, 2)
    assert _both(monkeypatch, lambda: rope(x, 5, out=out), plain) is out
    odd = torch.zeros(n, H, L, D + 1, dtype=dtype, device="cuda")[..., 1:]
    _both(monkeypatch, lambda: rope(x, 5, out=odd), False)


@pytest.mark.parametrize("fmt,dtype", [("fp16", torch.float32), ("bf16", torch.bfloat16), ("fp8", torch.float16),
                                       ("fp8_int4", torch.bfloat16)])
def test_write_read_attend(paged, monkeypatch, fmt, dtype):
    rope = paged.Rope(D, max_positions=64)
    k, v, q = (_randn(s, B, h, L, D, dtype=dtype) for s, h in ((3, H), (4, H), (5, H * G)))
    wide = _i(3, 1, 0, 9, 2, 5, 4, 9, 7, 6, -1, 9).view(3, 4)
    table = wide[:, :3]  # (rows are further apart than they are long)
    start = _i(0, 10, 30)

    def write(**kw):
        layer = paged.PagedLayer(9, H, D, PAGE, fmt)
        args = dict(k=k, v=v, table=table, start=start, q=q, rope=rope)
        args.update(kw)
        return [layer.write(**args), layer.k, layer.v, layer.k_exp, layer.v_scale]

    for kw in ({}, {"q": None}, {"rope": None}, {"n_new": _i(5, 0, 2)}, {"start": 2}, {"table": wide[:, :0]},
               {"n_new": _i(5, 0, 2), "q_out": torch.full_like(q, 7)}, {"q_out": torch.empty_like(q)},
               {"k": k[:, :, :0], "v": v[:, :, :0], "q": q[:, :, :0]}):
        _both(monkeypatch, lambda: write(**kw), True)
    _both(monkeypatch, lambda: write(table=wide[:, ::2]), False)
    _both(monkeypatch, lambda: write(n_new=_i(5, 1, 0, 1, 2, 1)[::2]), False)

    layer = paged.PagedLayer(9, H, D, PAGE, fmt)
    layer.write(k, v, table, start, rope=rope)
    lens = _i(5, 0, 35)
    for args, plain in (((), True), ((7,), True), ((7, torch.float32), True), ((0,), True), ((None, torch.bfloat16), True)):
        _both(monkeypatch, lambda: layer.read(table, lens, *args), plain)
    _both(monkeypatch, lambda: layer.read(wide[:, ::2], lens), False)

    one = q[:, :, :1].to(paged._NEW.get(fmt, torch.float16))
    for kw in ({}, {"max_len": 40}, {"max_len": 10 ** 6}, {"lens_add": -2}, {"scale": 0.3}, {"scale": 1}, {"return_lse": True},
               {"out": torch.empty_like(one, memory_format=torch.contiguous_format)}):
        _both(monkeypatch, lambda: layer.attend(one, table, lens, **kw), True)
    far = _i(*range(8)).repeat(B, 10)
    for kw in ({}, {"max_len": 900}):  # (split rows)
        _both(monkeypatch, lambda: layer.attend(one, far, _i(1200, 0, 700), **kw), True)
    _both(monkeypatch, lambda: layer.attend(one, wide[:, ::2], lens), False)
    _both(monkeypatch, lambda: layer.attend(one[:0], table[:0], lens[:0], return_lse=True), True)


def test_gradients_are_left_to_python(paged, monkeypatch):
    rope, x = paged.Rope(D, max_positions=64), _randn(1, B, H, L, D).requires_grad_()
    with pytest.raises(RuntimeError, match="requires grad"):
        rope(x)
    with torch.no_grad():
        _both(monkeypatch, lambda: rope(x, 3), False)


def test_threads_and_streams(paged):
    """Four threads, each on a stream of its own, with their own caches."""
    import threading

    rope = paged.Rope(D, max_positions=64)
    k, v, q = (_randn(s, B, h, 1, D) for s, h in ((3, H), (4, H), (5, H * G)))
    table, lens = _i(*range(9)).view(3, 3), _i(3, 20, 48)

    def run():
        layer = paged.PagedLayer(9, H, D, PAGE, "bf16")
        out = []
        for i in range(20):
            r = layer.write(k, v, table, lens - 1, q=q, rope=rope)
            out.append(layer.attend(r, table, lens))
        torch.cuda.current_stream().synchronize()
        return torch.stack(out)

    want = run()
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = run()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert all(g is not None and torch.equal(g, want) for g in got)
