"""What the paged cache's calls take and refuse beside plain arguments (GPU)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    import foveated_kv_amd
    from foveated_kv_amd import _lib, paged

    _lib.calls()
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return paged


def test_a_cuda_default_device(paged):
    """A program whose new tensors are the GPU's: the same table, cache and
    results."""
    def run():
        rope = paged.Rope(64, rot_dim=32, scaling={"kind": "ntk", "factor": 2.0}, max_positions=100)
        cache = paged.PagedKVCache(1, 2, 64, n_pages=8, max_seqs=2, max_tokens=64, page_size=16, rope=rope)
        g = torch.Generator(device="cpu").manual_seed(0)
        k, v, q = (torch.randn(2, h, n, 64, generator=g, device="cpu").half().cuda() for h, n in ((2, 5), (2, 5), (4, 5)))
        cache.extend([5, 3])
        cache.write(0, k, v)
        cache.extend(1)
        qr = cache.write(0, k[:, :, :1], v[:, :, :1], q=q[:, :, :1])
        return [rope.table, qr, cache.attend(0, qr), *cache.read(0)]

    want = run()
    with torch.device("cuda"):
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_chunk_for_sequences_of_different_lengths(paged):
    """A follow-up of five tokens for a sequence of 20 and a new one: what the
    model gets back is what each sequence gets alone."""
    from foveated_kv_amd import generate

    H, D, first, more = 2, 64, [20, 0], 5
    rope = paged.Rope(D, max_positions=64)
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(2, h, 25, D, generator=g).half().cuda() for h in (H, H, 2 * H))
    seen = []

    def attention(query, key, value, **kw):
        seen.append((query, key, value))
        return query

    def run(seqs):
        """The chunk of these sequences, each behind its own beginning."""
        cache = paged.PagedKVCache(1, H, D, n_pages=8, max_seqs=len(seqs), max_tokens=64, page_size=16, rope=rope)
        for i, b in enumerate(seqs):
            if first[b]:
                cache.extend(first[b], slice(i, i + 1))
                cache.write(0, k[b:b + 1, :, :first[b]], v[b:b + 1, :, :first[b]], seqs=slice(i, i + 1))
        part = [torch.cat([t[b:b + 1, :, first[b]:first[b] + more] for b in seqs]) for t in (k, v, q)]
        w, = generate.install_paged_attention(cache)
        generate._paged_state["original"], original = attention, generate._paged_state["original"]
        try:
            cache.extend(more)
            kk, vv = w.update_and_fetch(*part[:2])
            torch.nn.functional.scaled_dot_product_attention(part[2], kk, vv)
        finally:
            generate._paged_state["original"] = original
            generate.uninstall_paged_attention()
        return seen.pop()

    both = run([0, 1])
    assert both[1].shape == (2, H, 25, D)
    for b in (0, 1):
        n = first[b] + more
        alone = run([b])
        assert torch.equal(both[0][b], alone[0][0])
        for t, a in zip(both[1:], alone[1:]):
            assert torch.equal(t[b, :, :n], a[0]) and not bool(t[b, :, n:].any())


@pytest.mark.parametrize("yes,no", [(True, False), (1, 0), (np.True_, np.False_), ("yes", None)])
def test_return_lse_by_its_truth(paged, yes, no):
    layer = paged.PagedLayer(2, 1, 64, 16, "fp16")
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(2, 1)
    lens = torch.full((2,), 9, dtype=torch.int32, device="cuda")
    q = torch.ones(2, 4, 1, 64, dtype=torch.float16, device="cuda")
    out, lse = layer.attend(q, table, lens, return_lse=yes)
    assert out.shape == q.shape and lse.shape == (2, 4)
    assert torch.equal(layer.attend(q, table, lens, return_lse=no), out)


def test_a_forward_tangent_is_refused(paged):
    from torch.autograd import forward_ad

    rope, layer = paged.Rope(64, max_positions=8), paged.PagedLayer(1, 1, 64, 16, "fp16")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 1, 1, 64, dtype=torch.float16, device="cuda")
    with forward_ad.dual_level(), torch.no_grad():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: rope(d), lambda: rope(x, out=d), lambda: layer.write(d, x, table, 0),
                     lambda: layer.write(x, x, table, 0, q=d), lambda: layer.attend(d, table, lens)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert torch.equal(rope(x, 0), x)
    assert bool((layer.k == 0).all())


def _elements(t):
    """Storage offsets of a view's elements."""
    at = torch.zeros((), dtype=torch.int64) + t.storage_offset()
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return at.flatten()


def test_rows_that_share_memory(paged):
    """Random views of one buffer, read and written: refused where some element
    is in two rows (found here by listing them) unless the views are the same,
    and right where not."""
    import random

    from foveated_kv_amd import _lib

    D, rng, counts = 16, random.Random(11), {"same": 0, "apart": 0, "meet": 0}
    rope = paged.Rope(D, max_positions=64)
    table = rope.table.cpu().double()
    buf = torch.zeros(4096, dtype=torch.float32, device="cuda")

    def view(shape):
        kind = rng.choice(["nested", "nested", "any"])
        if kind == "any":
            strides = [8 * rng.randint(0, 20) for _ in shape]
        else:
            strides, order, s = [0] * 3, rng.sample(range(3), 3), D + 8 * rng.choice([0, 0, 1, 4])
            for d in order:
                strides[d] = s
                s = s * shape[d] + 8 * rng.choice([0, 0, 2])
        at = 8 * rng.randint(0, 60)
        if at + sum((n - 1) * s for n, s in zip(shape, strides)) + D > buf.numel():
            return view(shape)
        return torch.as_strided(buf, (*shape, D), (*strides, 1), at)

    for _ in range(400):
        shape = [rng.randint(1, 4) for _ in range(3)]
        x = view(shape)
        out = x if rng.random() < 0.2 else torch.as_strided(buf, x.shape, x.stride(), 8 * rng.randint(0, 60)) \
            if rng.random() < 0.5 and _elements(x).max() + 480 < buf.numel() else view(shape)
        ex, eo = _elements(x), _elements(out)
        inside = len(set(eo.tolist())) < len(eo)
        same = out.data_ptr() == x.data_ptr() and all(n == 1 or s == t for n, s, t in zip(shape, out.stride(), x.stride()))
        meet = inside or (not same and bool(torch.isin(eo, ex).any()))
        counts["meet" if meet else "same" if same else "apart"] += 1
        buf.copy_(torch.arange(4096))
        before = x.cpu().double()
        if meet:
            with pytest.raises((ValueError, _lib.FkvLibraryError), match="share memory"):
                rope(x, 3, out=out)
            assert torch.equal(buf, torch.arange(4096, device="cuda", dtype=torch.float32))
            continue
        rope(x, 3, out=out)
        c, s = (t[3:3 + shape[2]] for t in (table[:, 0], table[:, 1]))
        a, b = before[..., :D // 2], before[..., D // 2:]
        want = torch.cat([a * c - b * s, b * c + a * s], -1)
        # (one rounding to fp32 of a 64-bit sum of numbers up to 4096)
        assert bool(((out.cpu().double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -38).all())
    assert min(counts.values()) >= 40, counts


def test_heads_of_one_projection_in_place(paged):
    """q, k and v as one projection leaves them, interleaved in one buffer:
    nothing is shared, and q is rotated where it lies."""
    B, L, Hq, H, D = 2, 7, 4, 2, 64
    g = torch.Generator().manual_seed(1)
    for layout in ("blhd", "bhld"):
        x = torch.randn(B, L, Hq + 2 * H, D, generator=g).half().cuda()
        if layout == "bhld":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        q, k, v = (t.transpose(1, 2) for t in x.split([Hq, H, H], 2))
        rope, want = paged.Rope(D, max_positions=32), x.clone()
        layers = [paged.PagedLayer(B, H, D, 16, "fp16") for _ in range(2)]
        table = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1)
        qr = layers[0].write(k.clone(), v.clone(), table, 3, q=q.clone(), rope=rope)
        assert layers[1].write(k, v, table, 3, q=q, q_out=q, rope=rope) is q
        assert torch.equal(q, qr) and torch.equal(x[:, :, Hq:], want[:, :, Hq:])
        assert torch.equal(layers[0].k, layers[1].k) and torch.equal(layers[0].v, layers[1].v)


def test_attention_in_the_place_of_its_query(paged):
    layer = paged.PagedLayer(80, 2, 64, 16, "bf16")
    g = torch.Generator().manual_seed(2)
    layer.k.copy_(torch.randn(layer.k.shape, generator=g))
    layer.v.copy_(torch.randn(layer.v.shape, generator=g))
    q = torch.randn(2, 80, 1, 64, generator=g).bfloat16().cuda()
    table = torch.arange(80, dtype=torch.int32, device="cuda").view(2, 40)
    for n in (0, 100, 640):  # none, whole, split with two tiles of heads
        lens = torch.tensor([n, n // 2], dtype=torch.int32, device="cuda")
        want, x = layer.attend(q, table, lens), q.clone()
        assert torch.equal(layer.attend(x, table, lens, out=x), want) and torch.equal(x, want)


def test_what_a_layer_holds_is_fixed(paged):
    import copy

    layer = paged.PagedLayer(2, 1, 64, 16, "fp8")
    for name in ("k", "v", "k_exp", "v_scale", "page_size", "fmt"):
        with pytest.raises(AttributeError, match=f"{name} cannot be set"):
            setattr(layer, name, getattr(layer, name))
    with pytest.raises(TypeError):
        copy.deepcopy(layer)
    other = paged.PagedLayer.wrap("fp8", layer.k.clone(), layer.v.clone(), layer.k_exp.clone(), layer.v_scale.clone())
    x = torch.ones(1, 1, 1, 64, dtype=torch.float16, device="cuda")
    other.write(x, x, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 0)
    assert bool(other.k.any()) and not bool(layer.k.any())
