"""CPU tests of the text-decoding operators' host side at its edges."""

import math
from decimal import Decimal, localcontext

import pytest
import torch

from paged_model import turns_of

from pi05_infer import PagedKVCache, paged


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


@pytest.mark.parametrize("rotary,base,scaling,factor,original", [
    (2, 10000.0, None, 1.0, None), (512, 10000.0, None, 1.0, None), (128, 500000.0, "linear", 3.0, None),
    (64, 10000.0, "ntk", 8.0, None), (128, 10000.0, "yarn", 16.0, 8192), (8, 100.0, "yarn", 2.0, 4),
])
def test_table_is_rounded_once(rotary, base, scaling, factor, original):
    """Each entry is the whole number next to its fraction of a turn times 2^64, so that position 2^36 is still
    off by no more than 2^-29 turn."""
    exact, magnitude = paged._exact_frequencies(rotary, base, scaling, factor, original, 32.0, 1.0)
    assert magnitude == (0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0)
    with localcontext() as context:
        context.prec = 50
        for t, want in zip(paged._turns(exact), turns_of(rotary, base, scaling, factor, original), strict=True):
            assert abs(t - want * 2**64) <= Decimal("0.5000001")
