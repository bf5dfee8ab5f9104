"""A cache with sparse pages in generate_paged: prompts attend to everything before
them, however many tokens are left behind a beginning held in common; a drafting
cache may be sparse."""

import pytest
import torch

from test_gpu_paged_drafting import PROMPTS, SAME, _cache, _check_greedy, model  # noqa: F401
from test_gpu_paged_serving import fkv  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("left", [1, 2, 5])
def test_prompts_attend_to_all_pages(fkv, model, left):  # noqa: F811
    """The first token after prompts whose last `left` tokens follow a beginning held
    in common: that of a cache without sparse pages."""
    from foveated_kv_amd import generate

    m, tok = model
    text = (SAME * 3)[:160] + "abcde"[:left]
    prompts = [text, text[:-1] + "z"]
    ids = [tok.encode(p) for p in prompts]
    common = generate._common_tokens(ids, 16)
    assert common and len(ids[0]) - common == left
    logits = []
    for pages in (0, 2):
        cache = _cache(fkv, sparse_pages=pages)
        generate.install_paged_attention(cache)
        try:
            with torch.no_grad():
                logits.append(generate._prefill_paged(m, cache, ids, common, "cuda"))
        finally:
            generate.uninstall_paged_attention()
    assert torch.equal(logits[0], logits[1])


def test_sparse_drafts(fkv, model):  # noqa: F811
    from foveated_kv_amd import generate

    m, tok = model
    cache, drafts = _cache(fkv), _cache(fkv, sparse_pages=2)
    texts, stats = generate.generate_paged(m, tok, PROMPTS, cache, max_tokens=20, draft_model=m, draft_cache=drafts)
    _check_greedy(m, tok, texts, 20)
    assert stats["generated_tokens"] == [20] * 3
    with pytest.raises(ValueError, match="sparse_pages"):
        generate.generate_paged(m, tok, PROMPTS, drafts, max_tokens=20, draft_model=m, draft_cache=cache)
    assert cache.pages.free_pages == drafts.pages.free_pages == 60
