"""The paged cache as a program uses it: write, attend and read together over
many steps, prompts prefilled in chunks and in padded batches, whole models
served by ``generate_paged``, and a prompt's pages compressed into tiers."""

import numpy as np
import pytest
import torch

import _paged_ref as ref
import _tiny_lm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fkv():
    import foveated_kv_amd
    from foveated_kv_amd import _lib

    _lib.load()
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    assert foveated_kv_amd.is_available(), "libfkv.so loaded but no gfx950 device"
    return foveated_kv_amd


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("fmt,dtype", [("bf16", torch.bfloat16), ("fp8", torch.float16), ("fp8_int4", torch.bfloat16)])
def test_cache_run(fkv, fmt, dtype):
    """Three sequences: a padded prefill, decode steps, one sequence freed and
    begun anew in recycled pages, and after each step the attention of every
    layer against 64 bits over what the pages hold."""
    H, G, D, page, n_layers = 2, 4, 64, 16, 2
    rope = fkv.Rope(D, rot_dim=32, interleaved=True, max_positions=512)
    cache = fkv.PagedKVCache(n_layers, H, D, n_pages=24, max_seqs=3, max_tokens=160, page_size=page, fmt=fmt, rope=rope)
    t = rope.table.cpu().numpy()
    kept = [[None] * 3 for _ in range(n_layers)]  # rotated keys, values of each layer and sequence
    seed = [1000]

    def step(new, seqs=slice(0, 3)):
        cache.extend(new, seqs)
        n = cache.pages.lengths(seqs)
        starts = cache.pages.starts(seqs)
        L, B = max(a - b for a, b in zip(n, starts)), len(n)
        for i in range(n_layers):
            seed[0] += 3
            k, v, q = (_randn(seed[0] + j, B, L, h, D).to(dtype).cuda().transpose(1, 2)
                       for j, h in enumerate((H, H, H * G)))
            qr = cache.write(i, k, v, q, seqs=seqs)
            pos = np.array(starts)[:, None] + np.arange(L)
            k64, v64 = ref.rotate(ref.f64(k), pos, t, 32, True), ref.f64(v)
            q64 = ref.rotate(ref.f64(q), pos, t, 32, True)
            for j, b in enumerate(range(3)[seqs]):
                m = n[j] - starts[j]
                rows = [x[j, :, :m].astype(np.float32) for x in (k64, v64)]
                old = kept[i][b]
                kept[i][b] = rows if old is None else [np.concatenate([o, r], 1) for o, r in zip(old, rows)]
                got = ref.f64(qr[j, :, :m])
                assert (np.abs(got - q64[j, :, :m]) <= (ref.UNIT[dtype] + 2.0 ** -24) * np.abs(q64[j, :, :m]) * 1.001 +
                        ref.TINY[dtype]).all()
            rk, rv = cache.read(i, seqs, dtype=torch.float32)
            for j, b in enumerate(range(3)[seqs]):
                for got, want, name in zip((rk, rv), kept[i][b], "kv"):
                    g = got[j, :, :n[j]].cpu().double().numpy()
                    assert bool((got[j, :, n[j]:] == 0).all())
                    w = want.astype(np.float64)
                    if fmt == "bf16":
                        stands = torch.from_numpy(want).bfloat16().double().numpy()
                    elif fmt == "fp8" or name == "k":
                        c, e = ref.e4m3_encode(w)
                        stands = ref.e4m3_value(c) * 2.0 ** (e.astype(np.int64) - 127.0)[..., None]
                    else:
                        c, s, z = ref.int4_encode(w)
                        stands = c * s[..., None].astype(np.float64) + z[..., None].astype(np.float64)
                    assert (np.abs(g - stands) <= 2.0 ** -23 * np.abs(stands) + 2.0 ** -140).all()
            if L == 1:
                out = cache.attend(i, qr, seqs=seqs)
                layer = cache.layers[i]
                want, _, spread, ds = ref.attend(ref.f64(qr)[:, :, 0], ref.page_values(layer),
                                                 cache.pages.table[seqs].cpu().numpy(), n, page, 24, D ** -0.5)
                tol = ref.attend_bound(want, spread, ds, n, dtype)
                assert (np.abs(ref.f64(out)[:, :, 0] - want) <= tol).all()

    step([40, 1, 17])
    for _ in range(3):
        step(1)
    step([0, 30, 5])
    step(1)
    cache.free(0)
    for i in range(n_layers):
        kept[i][0] = None
    step(100, slice(0, 1))
    for _ in range(2):
        step(1)
    step(1, slice(1, 3))
    with pytest.raises(ValueError, match="made room for 1"):
        cache.write(0, *(torch.zeros(2, H, 2, D, dtype=dtype, device="cuda") for _ in range(2)), seqs=slice(1, 3))
    with pytest.raises(MemoryError):
        cache.extend(100)
    with pytest.raises(ValueError, match="one length"):
        cache.to_foveated()


def _model(fkv, n_layers=2, head_dim=64):
    return _tiny_lm.TinyLM(n_layers=n_layers, head_dim=head_dim, n_heads=8, n_kv_heads=2, seed=3).cuda().eval()


def _standard(model, ids, n):
    from foveated_kv_amd import generate

    caches = generate.make_prompt_cache(model)
    out = []
    with torch.no_grad():
        logits = model(torch.tensor([ids], device="cuda"), cache=caches)[:, -1]
        for _ in range(n):
            out.append(int(logits.argmax()))
            logits = model(torch.tensor([[out[-1]]], device="cuda"), cache=caches)[:, -1]
    return out


PROMPTS = ["the cat sat on the mat and then", "a dog", "x", "one two three four five six seven eight nine ten " * 4]


def test_generate_paged_equal_lengths(fkv):
    """A model that rotates by itself: the tokens of the standard cache."""
    from foveated_kv_amd import generate

    model, tok = _model(fkv), _tiny_lm.ByteTokenizer()
    prompts = [p[:30].ljust(30, "!") for p in PROMPTS]
    cache = fkv.PagedKVCache(2, 2, 64, n_pages=20, max_seqs=5, max_tokens=64, page_size=16)
    original = torch.nn.functional.scaled_dot_product_attention
    texts, stats = generate.generate_paged(model, tok, prompts, cache, max_tokens=12)
    assert torch.nn.functional.scaled_dot_product_attention is original
    assert texts == [tok.decode(_standard(model, tok.encode(p), 12)) for p in prompts]
    assert stats["stored_tokens"] == [42] * 4 and cache.pages.free_pages == 20
    assert stats["generated_tokens"] == [12] * 4 and stats["model_calls"] == 12
    text, _ = generate.generate_paged(model, tok, prompts[1], cache, max_tokens=5)
    assert text == tok.decode(_standard(model, tok.encode(prompts[1]), 5))


@pytest.mark.parametrize("fmt", ["fp16", "fp8"])
def test_generate_paged_rotated_by_the_cache(fkv, fmt, monkeypatch):
    """Prompts of different lengths (one token among them): the model leaves
    the rotation to the cache.  In 16-bit pages the tokens are the standard
    cache's; in quantised ones every sequence's run equals its run alone."""
    from foveated_kv_amd import generate

    model, tok = _model(fkv), _tiny_lm.ByteTokenizer()
    want = [_standard(model, tok.encode(p), 10) for p in PROMPTS]
    monkeypatch.setattr(_tiny_lm, "_rope", lambda x, offset, base=10000.0: x)
    rope = fkv.Rope(64, max_positions=512)

    def cache(n):
        return fkv.PagedKVCache(2, 2, 64, n_pages=40, max_seqs=n, max_tokens=256, page_size=16, fmt=fmt, rope=rope)

    texts, _ = generate.generate_paged(model, tok, PROMPTS, cache(4), max_tokens=10)
    if fmt == "fp16":
        assert texts == [tok.decode(w) for w in want]
    else:
        assert texts == [generate.generate_paged(model, tok, p, cache(1), max_tokens=10)[0] for p in PROMPTS]
    with pytest.raises(ValueError, match="different lengths"):
        generate.generate_paged(model, tok, PROMPTS, fkv.PagedKVCache(2, 2, 64, 40, 4), max_tokens=2)
    with pytest.raises(MemoryError):
        generate.generate_paged(model, tok, PROMPTS[3], fkv.PagedKVCache(2, 2, 64, 2, 1, page_size=16, rope=rope))
    # nothing of a failed run stays installed
    generate.install_paged_attention(cache(1))
    with pytest.raises(RuntimeError, match="installed"):
        generate.install_paged_attention(cache(1))
    with pytest.raises(RuntimeError, match="installed"):
        generate.install_fused_sdpa(fkv.FoveatedKVCache())
    generate.uninstall_paged_attention()


def test_generate_paged_stops_at_eos(fkv, monkeypatch):
    """A sequence that ends stops growing while the others go on; the last one
    to end ends the run."""
    from foveated_kv_amd import generate

    model, tok = _model(fkv), _tiny_lm.ByteTokenizer()
    want = [_standard(model, tok.encode(p), 14) for p in PROMPTS]
    monkeypatch.setattr(_tiny_lm, "_rope", lambda x, offset, base=10000.0: x)
    tok.eos_token_id = want[1][4]
    cut = [w[:w.index(tok.eos_token_id)] if tok.eos_token_id in w else w for w in want]
    n = [len(tok.encode(p)) for p in PROMPTS]
    cache = fkv.PagedKVCache(2, 2, 64, n_pages=40, max_seqs=4, max_tokens=256, page_size=16,
                             rope=fkv.Rope(64, max_positions=512))
    texts, stats = generate.generate_paged(model, tok, PROMPTS, cache, max_tokens=14)
    assert texts == [tok.decode(c) for c in cut] and len(cut[1]) <= 4
    assert stats["stored_tokens"] == [a + len(c) for a, c in zip(n, cut)]
    texts, stats = generate.generate_paged(model, tok, PROMPTS[1], cache, max_tokens=14)
    assert texts == tok.decode(cut[1]) and stats["model_calls"] == len(cut[1])
    assert cache.pages.free_pages == 40


def test_chunked_prefill_through_the_wrappers(fkv, monkeypatch):
    """A prompt fed in two chunks: the second one's queries attend to what
    the pages hold.  fp32 model, fp16 pages: logits as with whole prefill, up
    to the rounding of cached rows."""
    import torch.nn.functional as F

    from foveated_kv_amd import generate

    model, tok = _model(fkv), _tiny_lm.ByteTokenizer()
    ids = torch.tensor([tok.encode(PROMPTS[3])[:90]], device="cuda")

    def attention(x, cache):  # causal from the lower right corner, as a chunk needs
        q, k, v = x
        m = torch.ones(q.shape[2], k.shape[2], dtype=torch.bool, device="cuda").tril(k.shape[2] - q.shape[2])
        return F.scaled_dot_product_attention(q, k, v, attn_mask=m)

    H, D = 2, 64
    rope = fkv.Rope(D, max_positions=256)
    cache = fkv.PagedKVCache(1, H, D, n_pages=8, max_tokens=128, page_size=16, rope=rope)
    q, k, v = (_randn(5 + i, 1, H, 90, D).cuda() for i in range(3))
    with torch.no_grad():
        w = generate.install_paged_attention(cache, slice(0, 1))[0]
        try:
            outs = []
            for a, b in ((0, 50), (50, 90)):
                cache.extend(b - a)
                assert w.offset == a
                kk, vv = w.update_and_fetch(k[:, :, a:b], v[:, :, a:b])
                assert kk.shape[2] == b
                outs.append(attention((q[:, :, a:b], kk, vv), w))
            with pytest.raises(RuntimeError, match="call is missing"):
                w.update_and_fetch(k[:, :, :1], v[:, :, :1])
                w.update_and_fetch(k[:, :, :1], v[:, :, :1])
        finally:
            generate.uninstall_paged_attention()
        with pytest.raises(RuntimeError, match="not installed"):
            w.update_and_fetch(k[:, :, :1], v[:, :, :1])
    qr, kr = (ref.rotate(ref.f64(x), np.arange(90)[None], rope.table.cpu().numpy(), D, False) for x in (q, k))
    s = np.einsum("bhqd,bhkd->bhqk", qr, kr) * D ** -0.5
    s = np.where(np.tril(np.ones((90, 90), dtype=bool)), s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want = p @ ref.f64(v)
    # a cached key is off by 2^-11 of itself, a score by that of sum |q k|,
    # a weight by twice as much; a cached value by 2^-11; fp32 elsewhere
    ds = 2.0 ** -11 * np.einsum("bhqd,bhkd->bhqk", np.abs(qr), np.abs(kr)).max(-1)[..., None] * D ** -0.5
    tol = (2.02 * ds + 2.0 ** -11 + 2.0 ** -14) * (p @ np.abs(ref.f64(v)))
    assert (np.abs(ref.f64(torch.cat(outs, 2)) - want) <= tol).all()


def test_to_foveated(fkv):
    """Prompts prefilled into 16-bit pages, then into tiers: byte for byte the
    tiers of the same K and V handed over directly."""
    H, D, S = 2, 64, 700
    cfg = fkv.TierConfig()
    k, v = (_randn(20 + i, 2, H, S, D).half().cuda() for i in range(2))
    cache = fkv.PagedKVCache(1, H, D, n_pages=30, max_seqs=3, max_tokens=1024, page_size=64)
    cache.extend(S, slice(1, 3))
    cache.write(0, k, v, seqs=slice(1, 3))
    got = cache.to_foveated(cfg, seqs=slice(1, 3)).layers[0]
    plain = fkv.FoveatedKVCache(cfg)
    plain.update(k, v, 0)
    plain.compress()
    want = plain.layers[0]
    for name in ("near_k", "near_v", "far_k", "far_v", "far_v_scale", "far_v_zero", "near_valid", "archive_k", "far_idx"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    q = _randn(30, 2, H * 4, 1, D).half().cuda()
    assert torch.equal(got.attend_fused(q), want.attend_fused(q))


def test_refusals_on_the_device(fkv):
    from foveated_kv_amd import paged

    layer = paged.PagedLayer(4, 2, 64, 16, "fp16")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    kv = torch.zeros(1, 2, 3, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(1, 4, 1, 64, dtype=torch.float16, device="cuda")
    rope = paged.Rope(64, max_positions=8)
    bad = [
        (ValueError, lambda: layer.write(kv[:, :1], kv[:, :1], table, 0)),
        (ValueError, lambda: layer.write(kv, kv.float(), table, 0)),
        (TypeError, lambda: layer.write(kv.double(), kv.double(), table, 0)),
        (ValueError, lambda: layer.write(kv, kv, table.expand(2, -1), 0)),
        (TypeError, lambda: layer.write(kv, kv, table.long(), 0)),
        (TypeError, lambda: layer.write(kv, kv, table, torch.zeros(1, device="cuda"))),
        (ValueError, lambda: layer.write(kv, kv, table, torch.zeros(2, dtype=torch.int32, device="cuda"))),
        (ValueError, lambda: layer.write(kv, kv, table, torch.zeros(1, 3, dtype=torch.int32, device="cuda"))),
        (TypeError, lambda: layer.write(kv, kv, table, torch.zeros(1, dtype=torch.int32))),
        (ValueError, lambda: layer.write(kv, kv, table, 0, q=kv[:, :, :2])),
        (ValueError, lambda: layer.write(kv, kv, table, 0, q_out=kv)),
        (ValueError, lambda: layer.write(kv, kv, table, 0, rope=paged.Rope(128, max_positions=8))),
        (TypeError, lambda: layer.write(kv, kv, table, 0, n_new=lens.long())),
        (RuntimeError, lambda: layer.write(kv.clone().requires_grad_(), kv, table, 0)),
        (RuntimeError, lambda: rope(kv.clone().requires_grad_())),
        (ValueError, lambda: rope(kv[0])),
        (ValueError, lambda: rope(kv, torch.zeros(1, 2, dtype=torch.int32, device="cuda"))),
        (TypeError, lambda: rope(kv, torch.zeros(1, device="cuda"))),
        (ValueError, lambda: rope(kv, out=kv.float())),
        (TypeError, lambda: rope(kv.double())),
        (TypeError, lambda: layer.attend(q.float(), table, lens)),
        (TypeError, lambda: layer.attend(q.bfloat16(), table, lens)),
        (ValueError, lambda: layer.attend(q[:, :3], table, lens)),
        (ValueError, lambda: layer.attend(kv, table, lens)),
        (TypeError, lambda: layer.attend(q, table, lens.long())),
        (TypeError, lambda: layer.attend(q, table, 3)),
        (ValueError, lambda: layer.attend(q, table, lens, out=q.float())),
        (_lib_error(), lambda: layer.attend(q, table, lens, scale=float("nan"))),
        (ValueError, lambda: layer.read(table, lens, -1)),
        (TypeError, lambda: layer.read(table, lens, dtype=torch.int8)),
        (_lib_error(), lambda: paged.PagedLayer(4, 2, 96, 16)),
        (_lib_error(), lambda: paged.PagedLayer(4, 2, 64, 24)),
        (ValueError, lambda: paged.PagedLayer.wrap("fp8", layer.k, layer.v)),
        (ValueError, lambda: paged.PagedLayer.wrap("fp16", layer.k, layer.v[:2])),
    ]
    before = layer.k.clone()
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("accepted", i)
    assert torch.equal(layer.k, before)
    # nothing to do
    assert layer.attend(q[:0], table[:0], lens[:0]).shape == (0, 4, 1, 64)
    assert layer.read(table, lens, 0)[0].shape == (1, 2, 0, 64)
    layer.write(kv[:, :, :0], kv[:, :, :0], table, 0)
    assert bool((layer.attend(q, table[:, :0], lens) == 0).all())


def _lib_error():
    from foveated_kv_amd import _lib

    return _lib.FkvLibraryError


def test_pages_are_not_handed_out_in_a_capture(fkv):
    t = fkv.PageTable(4, 16, 2, 32)
    t.extend(3)
    x = torch.ones(4, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            x.add_(1)
            for call in (lambda: t.extend(1), lambda: t.reserve(20), lambda: t.free(0)):
                with pytest.raises(RuntimeError, match="outside of a capture"):
                    call()
        finally:
            graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        graph.replay()
    assert x.tolist() == [4.0] * 4
    assert t.lengths() == [3, 3] and t.free_pages == 2 and t.lens.tolist() == [3, 3]
    assert [t.table[b, 0].item() for b in range(2)] == [t.pages(b)[0] for b in range(2)]


def test_expanded_results_are_refused(fkv):
    from foveated_kv_amd import paged

    layer = paged.PagedLayer(4, 2, 64, 16, "fp16")
    rope = paged.Rope(64, max_positions=8)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    kv = torch.ones(1, 1, 3, 64, dtype=torch.float16, device="cuda").expand(-1, 2, -1, -1)
    for call in (lambda: rope(kv, 1, out=kv), lambda: layer.write(kv, kv, table, 0, q=kv, q_out=kv)):
        with pytest.raises(ValueError, match="share memory"):
            call()
    assert bool((layer.k == 0).all()) and bool((kv == 1).all())
    assert torch.equal(rope(kv, 1), rope(kv.contiguous(), 1))
