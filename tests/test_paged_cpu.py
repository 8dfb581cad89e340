"""CPU tests of the text-decoding operators' host side: refusals of the C ABI (reported before any device
work), struct layouts, and the rotary frequencies in 64 bits and fixed point."""

import ctypes
import math
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from conftest import REPO
from paged_model import angles

from pi05_infer import PagedKVCache, RopeFrequencies, _lib, paged, rope

BUF = (ctypes.c_char * (1 << 16))()
HERE = (ctypes.addressof(BUF) + 255) & ~255


def cache(**kw):
    c = paged.Pi05PagedCache(HERE, HERE, 2 * 16 * 64, 16 * 64, 64, HERE, HERE, HERE, HERE, 0, 8, 16, 2, 64, 3, 4, 4, HERE,
                             1 << 30)
    for n, v in kw.items():
        setattr(c, n, v)
    return ctypes.byref(c)


def call(name, *args):
    rc = paged._fn(name)(*args)
    return rc, _lib.last_error()


BAD_CACHES = [
    (dict(k_pages=None), 1), (dict(v_pages=None), 1), (dict(page_table=None), 1), (dict(counts=None), 1),
    (dict(dtype=2), 1), (dict(dtype=-1), 1), (dict(head_dim=60), 2), (dict(head_dim=264), 2), (dict(head_dim=0), 2),
    (dict(page_size=0), 2), (dict(num_pages=0), 2), (dict(batch=0), 2), (dict(n_kv_heads=0), 2),
    (dict(pages_per_seq=5), 2), (dict(pages_per_seq=1 << 28, table_pitch=1 << 28), 2), (dict(k_pages=HERE + 8), 3),
    (dict(page_stride=2 * 16 * 64 + 4), 3), (dict(row_stride=68), 3), (dict(workspace=None), 4),
    (dict(workspace_bytes=1000), 4), (dict(workspace=HERE + 16), 3), (dict(counts=HERE + 2), 3),
    (dict(weight=HERE + 1), 3), (dict(pos=HERE + 2), 3), (dict(page_table=HERE + 3), 3),
]


@pytest.mark.parametrize("kw,code", BAD_CACHES, ids=lambda x: str(x))
def test_bad_caches_are_refused(kw, code):
    a = paged.Pi05PagedAppend(HERE, HERE, 128, 64, 128, 64)
    a.tokens = 3
    t = paged.Pi05PagedAttention(HERE, HERE, None, None, 64, 64, 0, 0, 2, 1.0, 0, HERE, 1 << 30)
    for rc, text in (call("pi05_paged_append", cache(**kw), ctypes.byref(a), None),
                     call("pi05_paged_attention", cache(**kw), ctypes.byref(t), None),
                     call("pi05_paged_evict", cache(**kw), 8, 1, 1, None)):
        assert rc == code and text.startswith("paged_"), (rc, text)


def test_bad_arguments_are_refused():
    def append(rotary=None, **kw):
        a = paged.Pi05PagedAppend(HERE, HERE, 128, 64, 128, 64)
        a.tokens = 3
        if rotary is not None:
            a.rotary = ctypes.addressof(rotary)
        for n, v in kw.items():
            setattr(a, n, v)
        return call("pi05_paged_append", cache(weight=None) if "new_weight" in kw else cache(), ctypes.byref(a), None)[0]

    rot = paged.Pi05Rotary(HERE, 64, 0, 1.0)
    assert append(k=None) == 1 and append(v=None) == 1
    assert append(q=HERE, q_out=HERE, n_q_heads=4) == 1  # q, but nothing to rotate it by
    assert append(rot, q=HERE, n_q_heads=4) == 1         # no place for it
    assert append(rot, q=HERE, q_out=HERE, n_q_heads=0) == 2
    assert append(paged.Pi05Rotary(HERE, 66, 0, 1.0)) == 2 and append(paged.Pi05Rotary(HERE, 7, 0, 1.0)) == 2
    assert append(paged.Pi05Rotary(None, 64, 0, 1.0)) == 2
    assert append(tokens=4) == 2 and append(tokens=-1, cu_tokens=HERE) == 2
    assert append(new_weight=HERE) == 1
    assert append(tokens=0, cu_tokens=HERE) == 0         # nothing to do
    assert append(k=HERE + 1) == 3 and append(v=HERE + 1) == 3 and append(cu_tokens=HERE + 2) == 3
    assert append(paged.Pi05Rotary(HERE + 4, 64, 0, 1.0)) == 3
    assert append(k_token_stride=1 << 31) == 2 and append(v_head_stride=-64) == 2
    assert call("pi05_paged_append", cache(), None, None)[0] == 1

    def attend(c=None, **kw):
        a = paged.Pi05PagedAttention(HERE, HERE, None, None, 64, 64, 0, 0, 4, 1.0, 0, HERE, 1 << 30)
        for n, v in kw.items():
            setattr(a, n, v)
        return call("pi05_paged_attention", c or cache(), ctypes.byref(a), None)[0]

    assert attend(q=None) == 1 and attend(out=None) == 1
    assert attend(n_q_heads=3) == 2 and attend(n_q_heads=0) == 2
    assert attend(cache(weight=None), track=1) == 1
    assert attend(q=HERE + 2) == 3 and attend(q_head_stride=65) == 3 and attend(q_token_stride=65) == 3
    assert attend(out=HERE + 1) == 3 and attend(lse=HERE + 2) == 3
    big = cache(pages_per_seq=4096, table_pitch=4096)
    assert attend(big, scratch=None) == 4 and attend(big, scratch_bytes=64) == 4 and attend(big, scratch=HERE + 4) == 3
    assert call("pi05_paged_attention", cache(), None, None)[0] == 1

    for args in ((0, 0, 0), (4, -1, 0), (4, 0, -1), (4, 3, 2), (4, 2**31 - 1, 2)):
        assert call("pi05_paged_evict", cache(), *args, None)[0] == 2
    assert call("pi05_paged_evict", cache(weight=None), 4, 1, 1, None)[0] == 1
    assert call("pi05_paged_evict", cache(pos=None), 4, 1, 1, None)[0] == 1
    assert call("pi05_paged_evict", cache(), 64, 1, 1, None)[0] == 0  # 4 pages of 16: none can hold more

    def turn(x=HERE, out=HERE, dtype=0, tokens=2, heads=3, dim=64, xt=192, xh=64, ot=192, oh=64, pos=HERE, r=rot):
        a = paged.Pi05RopeArgs(x, out, pos, xt, xh, ot, oh, dtype, tokens, heads, dim, 0, 0)
        return call("pi05_rope", ctypes.byref(a), ctypes.byref(r) if r else None, None)[0]

    assert turn(x=None) == 1 and turn(out=None) == 1 and turn(pos=None) == 1 and turn(r=None) == 1
    assert turn(r=paged.Pi05Rotary(None, 64, 0, 1.0)) == 1 and turn(dtype=3) == 1
    assert turn(tokens=-1) == 2 and turn(heads=0) == 2 and turn(dim=62) == 2
    assert turn(r=paged.Pi05Rotary(HERE, 3, 0, 1.0)) == 2 and turn(r=paged.Pi05Rotary(HERE, 0, 0, 1.0)) == 2
    assert turn(ot=256) == 1  # in place, but with other strides
    assert turn(x=HERE + 1) == 3 and turn(out=HERE + 2, dtype=2) == 3 and turn(pos=HERE + 2) == 3
    assert turn(r=paged.Pi05Rotary(HERE + 4, 64, 0, 1.0)) == 3
    assert turn(out=HERE + 4096, xt=1 << 31) == 2 and turn(out=HERE + 4096, oh=-64) == 2
    assert turn(tokens=0) == 0


def test_sizes():
    ws, sc = paged._fn("pi05_paged_workspace_bytes"), paged._fn("pi05_paged_attention_scratch_bytes")
    assert ws(cache()) >= 16640 + 3 * 2 * (64 + 2) * 4 and ws(cache(batch=0)) == 0 and ws(None) == 0
    # a few short sequences need none; else fp32 partials, and scores of every row that there can be
    assert sc(cache(), 8, 0) == 0 and sc(cache(), 8, 1) == 0
    big = dict(pages_per_seq=4096, table_pitch=4096)
    plain, track = sc(cache(**big), 8, 0), sc(cache(**big), 8, 1)
    assert plain > 0 and track - plain >= 3 * 2 * 4096 * 16 * 4 * 4
    assert sc(cache(), 3, 0) == 0 and sc(None, 2, 0) == 0


def test_struct_layout_matches_header():
    types = (paged.Pi05Rotary, paged.Pi05RopeArgs, paged.Pi05PagedCache, paged.Pi05PagedAppend, paged.Pi05PagedAttention)
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"pi05_b200.h\"\nint main(void) {\n"
    for t in types:
        src += f'printf("{t.__name__} sizeof %zu\\n", sizeof({t.__name__}));\n'
        src += "".join(f'printf("{t.__name__} {f} %zu\\n", offsetof({t.__name__}, {f}));\n' for f, _ in t._fields_)
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        open(c, "w").write(src + "return 0;\n}\n")
        subprocess.run(["gcc", "-std=c99", "-I", os.path.join(REPO, "include"), c, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    by = {t.__name__: t for t in types}
    for line in out.splitlines():
        t, f, n = line.split()
        assert (ctypes.sizeof(by[t]) if f == "sizeof" else getattr(by[t], f).offset) == int(n), line


@pytest.mark.parametrize("packed,cls", [
    (paged._ROPE_ARGS, paged.Pi05RopeArgs), (paged._APPEND_ARGS, paged.Pi05PagedAppend),
    (paged._ATTEND_ARGS, paged.Pi05PagedAttention),
])
def test_packed_arguments_match_the_structs(packed, cls):
    """Each field, packed with a value of its own, comes back under its name."""
    values = list(range(1, len(cls._fields_) + 1))
    a = cls.from_buffer_copy(packed.pack(*values))
    assert packed.size == ctypes.sizeof(cls)
    assert [getattr(a, f) for f, _ in cls._fields_] == values


@pytest.mark.parametrize("rotary,base,scaling,factor,original", [
    (2, 10000.0, None, 1.0, None), (256, 10000.0, None, 1.0, None), (128, 500000.0, "linear", 4.0, None),
    (64, 10000.0, "ntk", 8.0, None), (128, 10000.0, "yarn", 16.0, 8192), (8, 100.0, "yarn", 2.0, 4),
])
def test_frequencies(rotary, base, scaling, factor, original):
    inv, mag = paged._pair_frequencies(rotary, base, scaling, factor, original, 32.0, 1.0)
    ref, ref_mag = angles(rotary, base, scaling, factor, original)
    assert np.allclose(inv, ref, rtol=1e-13, atol=0) and math.isclose(mag, ref_mag)
    turns = paged._turns(inv)
    assert all(0 <= t < 1 << 63 for t in turns)
    # angle of a far position in fixed point, wrapped, against 64 bits: 53-bit frequency, 2^-53 of the angle
    for pos in (1, 12345, 2**31 - 1, -77):
        for t, f in zip(turns, inv):
            got = (pos * t % (1 << 64)) / 2.0**64 * 2 * math.pi
            want = math.remainder(pos * f, 2 * math.pi)
            assert abs(math.remainder(got - want, 2 * math.pi)) <= abs(pos * f) * 2.0**-50 + 2.0**-30


@pytest.mark.parametrize("kw,text", [
    (dict(rotary_dim=3), "even"), (dict(rotary_dim=0), "even"), (dict(rotary_dim=514), "even"),
    (dict(rotary_dim=64, layout="pairs"), "layout"), (dict(rotary_dim=64, scaling="dynamic"), "scaling"),
    (dict(rotary_dim=64, base=1.0), "base"), (dict(rotary_dim=64, base=math.inf), "base"),
    (dict(rotary_dim=64, scaling="linear", factor=0.5), "factor"), (dict(rotary_dim=2, scaling="ntk", factor=2.0), "ntk"),
    (dict(rotary_dim=64, scaling="yarn", factor=2.0), "original_len"),
    (dict(rotary_dim=64, scaling="yarn", factor=2.0, original_len=10, beta_fast=1.0), "beta"),
    (dict(rotary_dim=64, device="cpu"), "CUDA device"),
])
def test_frequencies_refused(kw, text):
    with pytest.raises(ValueError, match=text):
        RopeFrequencies(**kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        rope(torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32), None)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache(k, k, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache.allocate(2, 16, 1, 64, 1, 2, device="cpu")
