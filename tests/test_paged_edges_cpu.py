"""CPU tests of the text-decoding operators' host side at its edges."""

import pytest
import torch

from pi05_infer import PagedKVCache


@pytest.mark.parametrize("name", ["k_pages", "v_pages", "page_table", "counts", "weight", "pos", "workspace"])
def test_tensors_of_a_cache_are_not_replaced(name):
    """The library keeps their addresses: another tensor would be ignored, and the first one's memory used after its end."""
    c = PagedKVCache.__new__(PagedKVCache)
    setattr(c, name, torch.zeros(2))  # as its constructor does
    with pytest.raises(AttributeError, match="write into it"):
        setattr(c, name, torch.ones(2))
    getattr(c, name).fill_(1)
    c.note = 1
    c.note = 2
