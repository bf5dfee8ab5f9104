"""Shared beginnings, drafted tokens and sparse attention as a program uses
them: one cache's sequences over many steps against 64 bits, and whole models
served by ``generate_paged``."""

import numpy as np
import pytest
import torch

import _paged_ref as ref
import _tiny_lm
from test_gpu_paged_serving import _model, _randn, fkv  # noqa: F401
from test_gpu_paged_tokens import _check as check_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,dtype", [("bf16", torch.bfloat16), ("fp8", torch.float16), ("fp8_int4", torch.bfloat16)])
def test_cache_run(fkv, fmt, dtype):  # noqa: F811
    """Four sequences: one prompt shared, each one's own tokens in padded
    batches, drafts refused and written again, one freed and begun anew; after
    each step every query's attention over what the pages hold."""
    H, G, D, page, n_layers = 2, 4, 64, 16, 2
    rope = fkv.Rope(D, max_positions=512)
    cache = fkv.PagedKVCache(n_layers, H, D, n_pages=40, max_seqs=4, max_tokens=160, page_size=page, fmt=fmt, rope=rope)
    seed = [2000]

    def step(new, seqs=slice(0, 4)):
        cache.extend(new, seqs)
        n, starts = cache.pages.lengths(seqs), cache.pages.starts(seqs)
        new = [a - b for a, b in zip(n, starts)]
        B, L = len(n), max(new)
        for i in range(n_layers):
            seed[0] += 3
            k, v, q = (_randn(seed[0] + j, B, L, h, D).to(dtype).cuda().transpose(1, 2) for j, h in enumerate((H, H, H * G)))
            q = cache.write(i, k, v, q, seqs=seqs)
            table, layer = cache.pages.table[seqs].cpu(), cache.layers[i]
            want = check_tokens(layer, q, table, n, new, shared=cache.pages.common_tokens(seqs), max_len=max(n))
            got = cache.attend_tokens(i, q, seqs)
            assert torch.equal(got, want)
            if L == 1:
                out = cache.attend(i, q, seqs)
                real = torch.tensor(new) > 0
                if cache.pages.common_tokens(seqs):
                    assert torch.equal(out[real], got[real])
                else:  # (by the one-token kernel, whose sums have another order)
                    w, _, spread, ds = ref.attend(ref.f64(q)[:, :, 0], ref.page_values(layer), table.numpy(), n, page, 40, D ** -0.5)
                    err = np.abs(ref.f64(out)[:, :, 0] - w)[real.numpy()]
                    assert (err <= ref.attend_bound(w, spread, ds, n, dtype)[real.numpy()]).all()
            with pytest.raises(ValueError, match="made room"):
                cache.attend_tokens(i, q[:, :, :1].expand(-1, -1, L + 1, -1), seqs)

    step(70, slice(0, 1))
    cache.share(0, 64, slice(1, 4))
    assert cache.pages.common_tokens() == 64
    step([0, 13, 1, 40])
    step(1)
    for back in ([3, 0, 4, 1], [2, 2, 2, 2], [0, 4, 3, 0]):
        step(4)
        cache.rollback(back)
    step([4, 2, 0, 1])
    cache.free(2)
    assert cache.pages.common_tokens() == 0
    step(30, slice(2, 3))
    step(1)
    step(3)
    cache.free(0)
    cache.share(3, 80, slice(0, 1))
    step([5, 1, 2, 3])
    assert cache.pages.common_tokens(slice(0, 1)) == 0
    for b in range(4):
        cache.free(b)
    assert cache.pages.free_pages == 40


SAME = "you are one of many readers of this long instruction, which all of you get first. "
PROMPTS = [SAME + "what is it?", SAME + "x", SAME + "tell me all about the cat on the mat, and then some more"]


@pytest.fixture
def model(fkv, monkeypatch):  # noqa: F811
    """A model whose rotation is left to the cache."""
    rotate = _tiny_lm._rope
    monkeypatch.setattr(_tiny_lm, "_rope", lambda x, offset, base=10000.0: x)
    m = _model(fkv)
    m.rotate = rotate
    return m, _tiny_lm.ByteTokenizer()


def _check_greedy(m, tok, texts, max_tokens):
    """Each token is the largest logit of the model with the standard fp32 cache
    after the same tokens, or so near to it that 16-bit rows may decide
    otherwise: queries, keys, values and results rounded by 2^-11 move a score
    of up to 8 by 2^-7, a weight by as much of itself, and the result by that of
    its terms, in each of two layers; the logits follow linearly: 2^-5 of the
    largest, with as much again for the norms between."""
    from foveated_kv_amd import generate

    patched, _tiny_lm._rope = _tiny_lm._rope, m.rotate
    try:
        for prompt, text in zip(PROMPTS, texts):
            ids, out = tok.encode(prompt), [int(t) for t in text.split()]
            assert tok.eos_token_id not in out and len(out) <= max_tokens
            with torch.no_grad():
                logits = m(torch.tensor([ids + out], device="cuda"), cache=generate.make_prompt_cache(m))[0, len(ids) - 1:]
            ends = out + ([tok.eos_token_id] if len(out) < max_tokens else [])
            for t, row in zip(ends, logits):
                assert float(row.max() - row[t]) <= 2.0 ** -4 * float(row.abs().max())
    finally:
        _tiny_lm._rope = patched


def _cache(fkv, fmt="fp16", n_layers=2, page=16, **kw):  # noqa: F811
    return fkv.PagedKVCache(n_layers, 2, 64, n_pages=60, max_seqs=3, max_tokens=256, page_size=page, fmt=fmt,
                            rope=fkv.Rope(64, max_positions=512), **kw)


def test_shared_prompts(fkv, model):  # noqa: F811
    from foveated_kv_amd import generate

    m, tok = model
    cache = _cache(fkv)
    texts, stats = generate.generate_paged(m, tok, PROMPTS, cache, max_tokens=20, share_prefix=True)
    _check_greedy(m, tok, texts, 20)
    assert stats["shared_tokens"] == len(tok.encode(SAME)) // 16 * 16 > 0 and cache.pages.free_pages == 60
    assert stats["stored_tokens"] == [len(tok.encode(p)) + 20 for p in PROMPTS]
    text, stats = generate.generate_paged(m, tok, PROMPTS[1], cache, max_tokens=4, share_prefix=True)
    assert stats["shared_tokens"] == 0 and stats["generated_tokens"] == [4] and len(text.split()) == 4


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("layers,n_draft,page", [(2, 4, 16), (1, 3, 32), (1, 7, 16), (1, 1, 16)])
def test_drafted_tokens(fkv, model, layers, n_draft, page, share):  # noqa: F811
    """Greedy: the model's own tokens, whatever the drafting model is (itself, or
    another one, whose pages have another size), in fewer calls."""
    from foveated_kv_amd import generate

    m, tok = model
    other = m if layers == 2 else _model(fkv, n_layers=1)
    cache, drafts = _cache(fkv), _cache(fkv, n_layers=layers, page=page)
    texts, stats = generate.generate_paged(m, tok, PROMPTS, cache, max_tokens=20, share_prefix=share, draft_model=other,
                                           draft_cache=drafts, n_draft=n_draft)
    _check_greedy(m, tok, texts, 20)
    assert stats["generated_tokens"] == [20] * 3 and 0 <= stats["accepted_tokens"] <= stats["drafted_tokens"]
    # (a round takes one token of each sequence at least)
    assert 4 <= stats["model_calls"] <= 19 if n_draft == 4 else stats["model_calls"] <= 19
    if layers == 2:
        assert stats["accepted_tokens"] > 0
    assert cache.pages.free_pages == drafts.pages.free_pages == 60


def test_drafting_stops_at_eos_and_max_tokens(fkv, model):  # noqa: F811
    from foveated_kv_amd import generate

    m, tok = model
    plain, _ = generate.generate_paged(m, tok, PROMPTS, _cache(fkv), max_tokens=20)
    tok.eos_token_id = int(plain[0].split()[7])
    for n in (20, 5, 1, 0):
        cache, drafts = _cache(fkv), _cache(fkv)
        texts, stats = generate.generate_paged(m, tok, PROMPTS, cache, max_tokens=n, draft_model=m, draft_cache=drafts)
        _check_greedy(m, tok, texts, n)
        assert cache.pages.free_pages == drafts.pages.free_pages == 60
    # no more room than each prompt and max_tokens take
    n = max(len(tok.encode(p)) for p in PROMPTS)
    caches = [fkv.PagedKVCache(2, 2, 64, n_pages=60, max_seqs=3, max_tokens=n + 9, page_size=16,
                               rope=fkv.Rope(64, max_positions=n + 9)) for _ in range(2)]
    texts, _ = generate.generate_paged(m, tok, PROMPTS, caches[0], max_tokens=9, draft_model=m, draft_cache=caches[1], n_draft=6)
    _check_greedy(m, tok, texts, 9)


def test_sampled_drafts(fkv, model):  # noqa: F811
    """Drawn tokens, of a drafting model equal to the target and of another one,
    over exact and quantised pages."""
    from foveated_kv_amd import generate

    m, tok = model
    torch.manual_seed(0)
    texts, stats = generate.generate_paged(m, tok, PROMPTS, _cache(fkv), max_tokens=12, temp=0.8, draft_model=m,
                                           draft_cache=_cache(fkv))
    assert stats["accepted_tokens"] > 0 and stats["generated_tokens"] == [12] * 3
    other = _model(fkv, n_layers=1)
    for fmt in ("fp8", "fp8_int4"):
        texts, stats = generate.generate_paged(m, tok, PROMPTS, _cache(fkv, fmt), max_tokens=12, temp=1.5, draft_model=other,
                                               draft_cache=_cache(fkv, n_layers=1), share_prefix=True)
        assert stats["generated_tokens"] == [12] * 3 and all(len(t.split()) == 12 for t in texts)


def test_sparse_pages(fkv, model):  # noqa: F811
    """All pages taken: the tokens of the whole attention.  Few: a run, and the
    layers' bounds are those of what they hold."""
    from foveated_kv_amd import generate

    m, tok = model
    for kw in ({}, {"share_prefix": True}):
        texts, _ = generate.generate_paged(m, tok, PROMPTS, _cache(fkv, sparse_pages=16), max_tokens=20, **kw)
        _check_greedy(m, tok, texts, 20)
    texts, stats = generate.generate_paged(m, tok, PROMPTS, _cache(fkv, "fp8", sparse_pages=3), max_tokens=20)
    assert stats["generated_tokens"] == [20] * 3
    cache = fkv.PagedKVCache(1, 2, 64, n_pages=9, max_seqs=2, max_tokens=64, page_size=16, sparse_pages=2)
    for n in ([20, 33], [1, 1], [3, 0]):
        cache.extend(n)
        k = _randn(sum(n), 2, 2, max(n), 64).half().cuda()
        cache.write(0, k, k)
    for b, n in enumerate(cache.pages.lengths()):
        keys = cache.read(0, slice(b, b + 1), torch.float32)[0][0].cpu()
        for i, p in enumerate(cache.pages.pages(b)):
            part = keys[:, 16 * i:min(16 * i + 16, n)]
            lo, hi = cache.layers[0].bounds[p].float().cpu().unbind(1)
            assert bool((lo <= part.amin(1)).all()) and bool((hi >= part.amax(1)).all())
            # (a step of bf16 at most)
            assert bool((part.amin(1) - lo <= 2.0 ** -7 * lo.abs()).all()) and bool((hi - part.amax(1) <= 2.0 ** -7 * hi.abs()).all())
