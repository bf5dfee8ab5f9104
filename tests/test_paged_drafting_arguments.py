"""What generate_paged refuses before it touches a GPU."""

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
