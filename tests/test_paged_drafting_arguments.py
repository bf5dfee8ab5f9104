"""What generate_paged refuses before it touches a GPU, and how many tokens its rounds
draft."""

from types import SimpleNamespace

import pytest
import torch

from foveated_kv_amd import PageTable, generate


class Tok:
    def encode(self, text):
        return [1, 2]


class Model:
    def parameters(self):
        return iter([torch.zeros(1)])


class Cache:
    rope = 1

    def __init__(self, sparse_pages=0):
        self.pages, self.sparse_pages = PageTable(4, 16, 2, 32, device="cpu"), sparse_pages


def test_no_drafting_for_a_cache_with_sparse_pages():
    """Verification attends to all pages, a step without drafts to few: the tokens
    would be neither model's."""
    with pytest.raises(ValueError, match="sparse_pages"):
        generate.generate_paged(Model(), Tok(), ["x"], Cache(3), draft_model=Model(), draft_cache=Cache())


@pytest.mark.parametrize("stands", [0, 1, 99])
@pytest.mark.parametrize("max_tokens,n_draft", [(1, 4), (2, 4), (7, 4), (12, 3), (12, 63)])
def test_no_token_is_drafted_that_cannot_be_taken(monkeypatch, stands, max_tokens, n_draft):
    """Each round drafts at most what a sequence may take beside the token that
    follows the drafts, and calls the drafting model for no other."""
    B, out, stored = 3, [[7], [7], [7]], [0, 0, 0]
    rounds, drafting = [], []

    def extend(n, seqs=None):
        for b, t in enumerate(n):
            stored[b] += t

    def rollback(n, seqs=None):
        for b, t in enumerate(n):
            stored[b] -= t

    pages = PageTable(64, 16, B, 256, device="cpu")
    cache = SimpleNamespace(layers=[], pages=pages, rope=1, extend=extend, rollback=rollback)

    def model(x, cache):
        return torch.zeros(B, x.shape[1], 10)

    def draft_model(x, cache):
        drafting.append(x.shape)
        return torch.zeros(B, 1, 10)

    def verify(target, probs, tokens, uniforms, n_draft):
        n, K = n_draft.tolist(), tokens.shape[1]
        rounds.append((list(n), [len(o) for o in out]))
        got = [min(t, stands) for t in n]
        rows = [[3] * (a + 1) + [-1] * (K - a) for a in got]
        return torch.tensor(rows), torch.tensor(got, dtype=torch.int32)

    monkeypatch.setattr(generate, "verify_drafts", verify)
    drafts = SimpleNamespace(layers=[], pages=pages, rope=1, extend=lambda n, seqs=None: None, rollback=lambda n, seqs=None: None)
    drafter = generate._Drafter(draft_model, drafts, n_draft)
    done = [False, False, False]
    generate._decode_drafted(model, cache, drafter, torch.tensor([7, 7, 7]), out, done, max_tokens, 0.0, None)
    assert [len(o) for o in out] == [max_tokens] * B and all(done)
    for n, have in rounds:
        assert all(t + 1 <= max_tokens - h for t, h in zip(n, have) if h < max_tokens) and max(n) <= n_draft
    # (a call for each drafted token, and one that stores the last, in rounds that draft)
    assert len(drafting) == sum(max(n) + 1 for n, _ in rounds if max(n) > 0)
    # all but the last token of each, which is the next round's
    assert stored == [max_tokens - 1] * B
