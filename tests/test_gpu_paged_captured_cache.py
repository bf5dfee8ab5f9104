"""The cache's own calls in captured graphs: replays follow the page table as it is
then, also where the sequences of the capture began alike or had as many new tokens."""

import pytest
import torch

from test_gpu_paged import _bits_equal, _flush, _randn
from test_gpu_paged_tokens import paged  # noqa: F401

pytestmark = pytest.mark.gpu

H, G, D, PAGE = 2, 3, 64, 16


def _cache(paged, fmt, B):  # noqa: F811
    return paged.PagedKVCache(1, H, D, 120, max_seqs=B, max_tokens=320, page_size=PAGE, fmt=fmt)


def _fill(cache, n, seq, seed):
    one = slice(seq, seq + 1)
    cache.extend(n, one)
    cache.write(0, _randn(seed, 1, H, n, D).bfloat16().cuda(), _randn(seed + 1, 1, H, n, D).bfloat16().cuda(), seqs=one)


def _graph(f):
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    s.synchronize()
    with torch.cuda.graph(g, stream=s):
        out = f()
    torch.cuda.synchronize()
    return g, out


def _near(a, b):
    # (two kernels' sums and a rounding each)
    assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -12).all())


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("L", [1, 3])
def test_sequences_that_no_longer_begin_alike(paged, fmt, L):  # noqa: F811
    _flush("captured", fmt, L)
    B = 4
    cache = _cache(paged, fmt, B)
    _fill(cache, 64, 0, 10)
    cache.share(0, 64, slice(1, B))
    for b in range(B):
        _fill(cache, 20 + b, b, 20 + 2 * b)
    k, v, q = (_randn(40 + i, B, n, L, D).bfloat16().cuda() for i, n in enumerate((H, H, H * G)))
    call = cache.attend if L == 1 else cache.attend_tokens

    def eager():
        table, lens = cache.pages.table, cache.pages.lens
        layer = cache.layers[0]
        return layer.attend(q, table, lens) if L == 1 else layer.attend_tokens(q, table, lens, n_new=cache.pages.new)

    cache.extend(L)
    cache.write(0, k, v)
    assert cache.pages.common_tokens() == 64
    g, out = _graph(lambda: call(0, q))
    for seed in (0, 1, 2):
        g.replay()
        torch.cuda.synchronize()
        _near(out, eager())
        _near(out, call(0, q))
        # other sequences in their places, with a beginning of their own
        for b in (0, 2) if seed == 0 else (1, 3) if seed == 1 else (0, 1, 2, 3):
            cache.free(b)
            _fill(cache, 50 + 31 * b + 7 * seed, b, 100 + 10 * b + seed)
        cache.extend(L)
        cache.write(0, k, v)
        torch.randn(1000, device="cuda").sum().item()
    g.replay()
    torch.cuda.synchronize()
    _near(out, eager())


def test_as_many_new_tokens_as_there_are_at_a_replay(paged):  # noqa: F811
    _flush("captured", "new")
    B, L = 3, 4
    caches = [_cache(paged, "bf16", B) for _ in range(2)]
    k, v, q = (_randn(60 + i, B, n, L, D).bfloat16().cuda() for i, n in enumerate((H, H, H * G)))
    for cache in caches:
        for b in range(B):
            _fill(cache, 30 + 17 * b, b, 70 + 2 * b)
        cache.extend(L)

    def step(cache):
        x = cache.write(0, k, v, q)
        return cache.attend_tokens(0, x)

    captured, plain = caches
    g, out = _graph(lambda: step(captured))
    g.replay()
    torch.cuda.synchronize()
    _bits_equal(out, step(plain), "as captured")
    for new in ([4, 0, 2], [1, 4, 3], [4, 4, 4]):
        for cache in caches:
            cache.extend(new)
        g.replay()
        torch.cuda.synchronize()
        want = step(plain)
        for b, n in enumerate(new):
            _bits_equal(out[b, :, :n], want[b, :, :n], f"{new}")
        for x, y in zip(captured.read(0), plain.read(0)):
            _bits_equal(x, y, "what is stored")


def test_sparse_steps(paged):  # noqa: F811
    _flush("captured", "sparse")
    cache = paged.PagedKVCache(1, H, D, 120, max_seqs=2, max_tokens=320, page_size=PAGE, fmt="bf16", sparse_pages=4)
    for b in range(2):
        _fill(cache, 150 + 40 * b, b, 80 + 2 * b)
    q = _randn(90, 2, H * G, 1, D).bfloat16().cuda()
    g, out = _graph(lambda: cache.attend(0, q))
    for n in (5, 33):
        g.replay()
        torch.cuda.synchronize()
        _bits_equal(out, cache.attend(0, q), "replay")
        for b in range(2):
            _fill(cache, n, b, 200 + n + b)
