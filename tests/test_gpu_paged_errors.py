"""The paged cache's calls when something fails that is not an argument: the
call's own errors are raised and its work is not done twice, another call's are
left to that one."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

B, H, L, D, PAGE = 2, 2, 3, 64, 16


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.calls()
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def _calls(paged, dtype=torch.float16):
    """name -> the call in place, and what it writes."""
    x = torch.randn(B, H, L, D, generator=torch.Generator().manual_seed(1)).to("cuda", dtype)
    rope = paged.Rope(D, max_positions=32)
    layer = paged.PagedLayer(B, H, D, PAGE, "fp16")
    table = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1)
    lens = torch.full((B,), 5, dtype=torch.int32, device="cuda")
    out = torch.zeros(B, H, 1, D, dtype=dtype, device="cuda")
    q, kv = x.clone(), x.clone()
    return {
        "fkv_rope_apply": (lambda: rope(x, 3, out=x), x),
        "fkv_paged_write": (lambda: layer.write(kv, kv, table, 2, q=q, q_out=q, rope=rope), q),
        "fkv_paged_read": (lambda: layer.read(table, lens), layer.k),
        "fkv_paged_attn": (lambda: layer.attend(x[:, :, :1], table, lens, out=out), out),
    }


ENTRIES = ["fkv_rope_apply", "fkv_paged_write", "fkv_paged_read", "fkv_paged_attn"]


@pytest.fixture
def stub():
    """Binds the compiled calls to an entry point that counts its calls and
    returns ``code``."""
    from foveated_kv_amd import _lib

    lib, calls, kept = _lib.load(), _lib.calls(), []

    def address(f):
        return ctypes.cast(f, ctypes.c_void_p).value

    names = ["fkv_rope_apply", "fkv_paged_write", "fkv_paged_read", "fkv_paged_attn_workspace", "fkv_paged_attn"]

    def bind(name, code):
        seen = []
        sig = _lib.SIGNATURES[name]
        f = ctypes.CFUNCTYPE(sig[0], *sig[1])(lambda *args: seen.append(1) or code)
        kept.append(f)
        calls.bind(*(address(f if n == name else getattr(lib, n)) for n in names), _lib.check)
        return seen

    yield bind
    calls.bind(*(address(getattr(lib, n)) for n in names), _lib.check)


@pytest.mark.parametrize("code", [-2, -3])
@pytest.mark.parametrize("name", ENTRIES)
def test_a_failed_call_is_raised_and_not_made_again(paged, stub, name, code):
    from foveated_kv_amd import _lib

    call, target = _calls(paged)[name]
    before = target.clone()
    seen = stub(name, code)
    with pytest.raises(_lib.FkvLibraryError, match=rf"{name} failed \({code}\)"):
        call()
    assert len(seen) == 1 and torch.equal(target, before)


@pytest.mark.parametrize("name", ENTRIES)
def test_a_refusal_is_left_to_python(paged, stub, name):
    call, _ = _calls(paged)[name]
    seen = stub(name, -1)
    call()
    assert len(seen) == 1


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("name", ENTRIES)
def test_an_error_that_was_there_before(paged, monkeypatch, name, compiled):
    """Another call's pending error is no failure of this one, and stays for
    the program to find."""
    from foveated_kv_amd import _lib

    class Left:
        def __getattr__(self, name):
            return lambda *args: NotImplemented

    want, target = _calls(paged)[name]
    want()
    expected = target.clone()
    call, target = _calls(paged)[name]
    call_again, _ = _calls(paged)[name]
    call_again()  # (everything that allocates or loads code has done so)
    torch.cuda.synchronize()
    if not compiled:
        monkeypatch.setattr(_lib, "calls", Left)
    lib = ctypes.CDLL(_lib.LIB_PATH)  # (its HIP runtime is torch's)
    assert lib.hipSetDevice(1 << 20) != 0
    pending = lib.hipPeekAtLastError()
    assert pending != 0
    try:
        call()
        left = lib.hipPeekAtLastError()
    finally:
        lib.hipGetLastError()
    torch.cuda.synchronize()
    assert left == pending and torch.equal(target, expected)
