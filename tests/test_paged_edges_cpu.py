"""CPU tests of the text-decoding operators' host side at its edges."""

import ctypes
import math
from decimal import Decimal, localcontext

import numpy as np
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


def test_sizes_go_by_the_pool():
    """Scratch and workspace behind tables for 131072 rows, 256 sequences, 8 heads, over 65536 pages of 16 rows."""
    def sizes(weight=16, **kw):
        shape = dict(num_pages=65536, page_size=16, n_kv_heads=8, head_dim=128, batch=256, pages_per_seq=8192) | kw
        c = paged.Pi05PagedCache(dtype=0, weight=weight, pos=weight, table_pitch=shape["pages_per_seq"], **shape)
        at = ctypes.byref(c)
        scratch = [paged._fn("pi05_paged_attention_scratch_bytes")(at, 32, track) for track in (0, 1)]
        return paged._fn("pi05_paged_workspace_bytes")(at), scratch[1] - scratch[0]

    slots = 65536 * 16 * 8
    lists, scores = sizes()
    assert 4 * slots <= lists < 4 * slots + (1 << 16)  # 34 MB; by the table it was 1.07 GB
    assert 16 * slots <= scores < 16 * slots + 256 * 8 * 3 * 64 * 16 + (1 << 16)  # 138 MB; 4.3 GB
    assert sizes(weight=None)[0] < 1 << 15
    lists, scores = sizes(num_pages=64)  # small pools: never less than 64 MB where the table asks for more
    assert lists < 1 << 17 and 60 << 20 < scores < 65 << 20
    lists, scores = sizes(pages_per_seq=16, num_pages=1 << 20)  # short tables over a large pool: by the table
    assert lists < 4 * 256 * 8 * 256 + (1 << 16) and scores < 16 * 256 * 8 * (256 + 128) + (1 << 16)


def test_frequencies_of_other_number_types():
    want = paged._exact_frequencies(64, 500000.0, "ntk", 8.0, None, 32.0, 1.0)
    for of in (int, np.float32, np.float64):
        assert paged._exact_frequencies(64, of(500000), "ntk", of(8), None, 32.0, 1.0) == want
