"""What the paged cache's calls take and refuse beside plain arguments (CPU)."""

import ctypes

import pytest
import torch

from foveated_kv_amd import Rope, _lib, paged
from test_paged import SCALINGS


@pytest.mark.parametrize("scaling", SCALINGS)
def test_rope_under_another_default_device(scaling):
    """The frequencies are host memory whatever torch's default device is."""
    want = Rope(64, scaling=scaling, max_positions=40, device="cpu").table
    with torch.device("meta"):
        inv, _ = paged._frequencies(64, 10000.0, scaling)
        assert inv.device.type == "cpu" and inv.is_contiguous()
        got = Rope(64, scaling=scaling, max_positions=40, device="cpu").table
    assert got.device.type == "cpu" and torch.equal(got, want)


class _Recorded:
    """A cache whose pages are handed out and whose layers only note calls."""

    rope, layers = None, [None]

    def __init__(self, fails=False):
        self.pages, self.done, self.fails = paged.PageTable(8, 16, 2, 64, device="cpu"), [], fails

    def write(self, *args, **kw):
        self.done.append("write")
        if self.fails:
            raise RuntimeError("no write")

    def read(self, layer, seqs, dtype):
        self.done.append("read")
        return "k", "v"


def test_chunks_at_different_beginnings():
    """Whether there is something to read back is a matter of every sequence's
    beginning, which the host knows."""
    from foveated_kv_amd import generate

    cache, kv = _Recorded(), torch.zeros(2, 1, 5, 64)
    w, = generate.install_paged_attention(cache)
    try:
        cache.pages.extend(5)
        assert w.offset == 0 and w.update_and_fetch(kv, kv) == (kv, kv) and cache.done == ["write"]
        torch.nn.functional.scaled_dot_product_attention(kv, kv, kv)
        cache.pages.free(1)
        cache.pages.extend(5)
        assert w.offset.tolist() == [5, 0]
        assert w.update_and_fetch(kv, kv) == ("k", "v") and cache.done == ["write", "write", "read"]
        torch.nn.functional.scaled_dot_product_attention(kv, kv, kv)
    finally:
        generate.uninstall_paged_attention()


def test_a_failed_update_leaves_nothing_pending():
    from foveated_kv_amd import generate

    cache, kv = _Recorded(fails=True), torch.zeros(2, 1, 5, 64)
    w, = generate.install_paged_attention(cache)
    try:
        for _ in range(2):
            with pytest.raises(RuntimeError, match="no write"):
                w.update_and_fetch(kv, kv)
        torch.nn.functional.scaled_dot_product_attention(kv[:, :, :2], kv, kv)  # (another attention)
    finally:
        generate.uninstall_paged_attention()


def test_a_forward_tangent_is_refused():
    from torch.autograd import forward_ad

    x = torch.zeros(1, 2, 3, 64)
    with forward_ad.dual_level():
        paged._on(-1, "x", x)
        with pytest.raises(RuntimeError, match="tangent"):
            paged._on(-1, "x", forward_ad.make_dual(x, torch.ones_like(x)))


# ---------------------------------------------------------------------------
# rows that share memory (entry points refuse them before any launch)
# ---------------------------------------------------------------------------

def _entry(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    assert rc == _lib.FKV_EINVAL, rc
    return lib.fkv_last_error().decode()


def _rows(at, sb, sh, sl):
    return ctypes.byref(_lib.RowsC(at, sb, sh, sl))


def test_results_that_share_memory_are_refused():
    """B, H, L, D = 2, 3, 4, 64 of fp16; addresses and strides in one buffer
    that is never touched."""
    at = 1 << 20
    rope = ctypes.byref(_lib.RopeC(at, 4, 64, 0))
    pos = ctypes.byref(_lib.PositionsC(None))
    x = (at, 768, 256, 64)
    for out, word in [((at, 768, 256, 0), "rows of out"), ((at, 768, 256, 56), "rows of out"), ((at, 512, 256, 64), "rows of out"),
                      ((at, 256, 256, 64), "rows of out"), ((at, 768, 256, -32), "rows of out"),
                      ((at + 128, *x[1:]), "out, which is not x"), ((at + 16, *x[1:]), "out, which is not x"),
                      ((at - 2 * 704, *x[1:]), "out, which is not x"), ((at, 768, 64, 192), "out, which is not x"),
                      ((at + 2 * 1472, 64, 128, 512), "out, which is not x"), ((at + 384, 768, 256, -64), "out, which is not x")]:
        msg = _entry("fkv_rope_apply", rope, _rows(*x), _rows(*out), 0, 2, 3, 4, 64, pos, None)
        assert word in msg and "share memory" in msg, (out, msg)
    pages = ctypes.byref(_lib.PagesC(at, at, None, None, 2, 16, 3, 64, 0))
    far = (at + (1 << 18), 768, 256, 64)
    for q, q_out, k, v, word in [(x, (at + 128, *x[1:]), far, far, "q_out, which is not q"), (x, x, x, far, "q_out and k"),
                                 (x, x, far, x, "q_out and v"), (far, x, (at + 2 * 768, *x[1:]), far, "q_out and k"),
                                 (far, (at, 768, 256, 32), far, far, "rows of q_out")]:
        msg = _entry("fkv_paged_write", pages, _rows(*k), _rows(*v), 0, 2, 4, at, 1, 1, pos, None, None, _rows(*q),
                     _rows(*q_out), 3, None)
        assert word in msg and "share memory" in msg, (word, msg)
    for q, out in [((at, 192, 64, 0), at + 128), ((at, 384, 128, 0), at), ((at, 192, 64, 0), at - 2 * 320)]:
        msg = _entry("fkv_paged_attn", pages, _rows(*q), 0, 3, 2, at, 1, 1, at, 0, 16, 1.0, out, None, None, 0, None)
        assert "out, which is not the query" in msg


# ---------------------------------------------------------------------------
# objects
# ---------------------------------------------------------------------------

def test_what_a_rope_is_made_for_is_fixed():
    """Its calls know the table's address: another table, or another way to
    pair, would have been ignored."""
    import copy

    rope = Rope(64, max_positions=8, device="cpu")
    for name, value in (("table", rope.table * 0), ("interleaved", True), ("rot_dim", 32), ("head_dim", 128)):
        with pytest.raises(AttributeError, match=f"{name} cannot be set"):
            setattr(rope, name, value)
        with pytest.raises(AttributeError):
            setattr(copy.copy(rope), name, value)
    with pytest.raises(TypeError):  # (a copy of the table at another address)
        copy.deepcopy(rope)
    assert not rope.interleaved and rope.table.any()
    rope.note = "mine"  # (a program's own)


def test_numbers_of_tokens():
    """Anything that is an integer, or a sequence of them."""
    import numpy as np

    t = paged.PageTable(16, 16, 2, 100, device="cpu")
    for n, lens in ((np.int64(3), [3, 3]), (torch.tensor(2), [5, 5]), (np.array([1, 0]), [6, 5]), (torch.tensor([0, 4]), [6, 9]),
                    ((1, np.int32(1)), [7, 10]), (True, [8, 11])):
        t.extend(n)
        assert t.lengths() == lens and t.lens.tolist() == lens
    t.reserve(np.int32(40))
    assert [len(t.pages(b)) for b in (0, 1)] == [3, 3]
    for bad in (1.5, None, torch.tensor(0.5)):
        with pytest.raises(TypeError):
            t.extend(bad)
    for bad in ([1, 1, 1], torch.tensor([1])):
        with pytest.raises(ValueError, match="for 2 sequences"):
            t.extend(bad)
    assert t.lengths() == [8, 11]


def test_a_cache_does_not_grow_past_its_rotary_table():
    """Keys there would be NaN, and with them all that the sequence attends
    to."""
    cache = paged.PagedKVCache.__new__(paged.PagedKVCache)
    cache.pages = paged.PageTable(8, 16, 2, 64, device="cpu")
    cache.rope = Rope(64, max_positions=20, device="cpu")
    cache.extend([20, 3])
    for n, seqs in ((1, None), ([1, 0], None), ([0, 18], None), (1, slice(0, 1))):
        with pytest.raises(ValueError, match="20 positions"):
            cache.extend(n, seqs)
        assert cache.pages.lengths() == [20, 3] and cache.pages.starts() == [0, 0]
    cache.extend([0, 17])
    cache.extend(0)
    assert cache.pages.lengths() == [20, 20]
    cache.rope = None
    cache.extend(1)
    with pytest.raises(MemoryError):
        cache.extend(44)
