"""GPU tests of the text-decoding operators (rotary positions, paged cache append, attention, eviction)
against ``paged_model.py`` in 64 bits.

Tolerances.  u = eps / 2 of the element type, one rounding to it; f = 2^-24, one fp32 rounding.

* rotation: cos and sin are within 2 ulp of fp32 (4 f) of the 64-bit ones, their product with the
  magnitude, the two products and the sum add 4 f: 8 f (|a| + |b|) magnitude, then u of the result.
* scores: dim products and sums in fp32, 2 dim f of sum |q| |k| (the matrix unit may truncate, hence 2
  rather than 1), scaled: e = 2 dim f reach + 4 f |score|, where |score| <= reach.  A probability is then
  off by the factor 1 + 2 e + 16 f (exp2 to 2 ulp, its argument's rounding, the sum, the division).
* output: u of the result, and u of each probability rounded to the element type for the second
  product (fp16 below 2^-14 instead 2^-25 each): (u + 2 e + 16 f) sum p |v| + u |out|.
* moved rows, positions and counts: exact.
"""

import numpy as np
import pytest
import torch

from paged_model import Cache, rotate

from pi05_infer import PagedKVCache, RopeFrequencies, rope

pytestmark = pytest.mark.gpu

F = 2.0**-24
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def u(dtype):
    return torch.finfo(dtype).eps / 2


def np64(t):
    return t.detach().double().cpu().numpy()


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(*shape, dtype=BF, g=None, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


def check_rope(y, x, positions, rotary, layout, back=False, **kw):
    ref, size = rotate(np64(x), positions.cpu().numpy(), rotary, layout, back, **kw)
    tol = 8 * F * size
    tol = tol + (u(y.dtype) if y.dtype != FP else 0) * (np.abs(ref) + tol) + (2.0**-25 if y.dtype == HF else 0)
    err = np.abs(np64(y) - ref)
    assert (err <= tol).all(), (err - tol).max()
    assert (np64(y)[..., rotary:] == np64(x)[..., rotary:]).all()  # the rest passes through


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rotary", [
    (1, 1, 2, 2), (1, 9, 256, 256), (5, 3, 72, 72), (33, 4, 128, 64), (7, 2, 80, 10), (300, 5, 96, 6), (3, 2, 9, 4),
    (70, 33, 64, 48), (2, 1, 512, 512),
])
def test_rope(dtype, layout, tokens, heads, dim, rotary):
    g = gen(tokens)
    x = rnd(tokens, heads, dim, dtype=dtype, g=g)
    pos = torch.randint(-5000, 5000, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    f = RopeFrequencies(rotary, layout=layout)
    y = rope(x, pos, f)
    check_rope(y, x, pos, rotary, layout)
    assert torch.equal(rope(x, pos.long(), f), y)
    check_rope(rope(x, pos, f, transpose=True), x, pos, rotary, layout, back=True)
    z = x.clone()
    assert rope(z, pos, f, out=z) is z and torch.equal(z, y)  # in place


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rotary", [4, 8, 12, 20, 36, 40])
@pytest.mark.parametrize("skip,dim,room", [(0, 40, 0), (4, 40, 4), (2, 42, 2), (1, 41, 0), (0, 40, 1)])
def test_rope_words(dtype, layout, rotary, skip, dim, room):
    """Every word that pairs, strides and the first row's address allow gives the same values."""
    n, h = 19, 3
    buf = rnd(n, h * dim + skip + room, dtype=dtype, g=gen(rotary))
    x = buf[:, skip : skip + h * dim].unflatten(1, (h, dim))
    pos = torch.arange(n, device="cuda", dtype=torch.int32) * 31 - 100
    f = RopeFrequencies(rotary, layout=layout)
    out = torch.full_like(buf, 7.0)
    y = rope(x, pos, f, out=out[:, skip : skip + h * dim].unflatten(1, (h, dim)))
    check_rope(y, x, pos, rotary, layout)
    assert (out[:, :skip] == 7).all() and (out[:, skip + h * dim :] == 7).all()
    assert torch.equal(rope(x.contiguous(), pos, f), y)


@pytest.mark.parametrize("kw", [
    dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0, base=500000.0),
    dict(scaling="yarn", factor=16.0, original_len=8192),
    dict(scaling="yarn", factor=2.0, original_len=4, base=100.0),  # every pair below one turn
])
def test_rope_scaled_and_far(kw):
    """Positions up to 2^31 - 1: the angle keeps its 2^-33 turn, and with it the tolerance of near ones; the
    64-bit reference's own angle is good to 2^31 2^-53 rad, below f."""
    g = gen(1)
    pos = torch.tensor([0, 1, 8191, 131072, 10**6 + 1, 2**31 - 1, -(2**31)], device="cuda", dtype=torch.int32)
    x = rnd(len(pos), 3, 64, dtype=FP, g=g)
    f = RopeFrequencies(64, layout="interleaved", **kw)
    m = dict(kw)
    if "original_len" in m:
        m["original"] = m.pop("original_len")
    y = rope(x, pos, f)
    ref, size = rotate(np64(x), pos.cpu().numpy(), 64, "interleaved", **m)
    # the frequencies are 64-bit floats on both sides: 2^-52 of an angle of up to 2^31 rad
    tol = (8 * F + np.abs(np64(pos))[:, None, None] * 2.0**-51) * size
    assert (np.abs(np64(y) - ref) <= tol).all()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_rope_views(dtype):
    """q and k heads inside q|k|v rows, read and written in place; v and what is beside it stay."""
    g = gen(2)
    qkv = rnd(40, 10, 128, dtype=dtype, g=g)
    was = qkv.clone()
    pos = torch.arange(40, device="cuda")
    f = RopeFrequencies(128)
    rope(qkv[:, :9], pos, f, out=qkv[:, :9])
    check_rope(qkv[:, :9], was[:, :9], pos, 128, "half")
    assert torch.equal(qkv[:, 9], was[:, 9])
    # heads first in memory, rows off a 16-byte boundary
    odd = rnd(5, 41, 131, dtype=dtype, g=g)[:, 1:, 3:].transpose(0, 1)
    check_rope(rope(odd, pos, f), odd, pos, 128, "half")
    out = torch.zeros(40, 7, 130, dtype=dtype, device="cuda")
    rope(odd, pos, f, out=out[:, 1:6, 1:129])
    check_rope(out[:, 1:6, 1:129], odd, pos, 128, "half")
    assert (out[:, 0] == 0).all() and (out[:, 6] == 0).all() and (out[..., 0] == 0).all() and (out[..., 129] == 0).all()


def test_rope_empty():
    x = torch.empty(0, 4, 64, dtype=BF, device="cuda")
    assert rope(x, torch.empty(0, dtype=torch.int32, device="cuda"), RopeFrequencies(64)).shape == (0, 4, 64)


@pytest.mark.parametrize("layout,scaling", [("half", None), ("interleaved", "yarn")])
def test_rope_gradient(layout, scaling):
    """Against the formula (the transposed rotation), a broadcast incoming gradient, and differences."""
    g = gen(3)
    kw = dict(scaling=scaling, factor=4.0, original_len=64) if scaling else {}
    f = RopeFrequencies(20, layout=layout, **kw)
    if scaling:
        kw["original"] = kw.pop("original_len")
    pos = torch.randint(0, 1000, (11,), device="cuda", generator=g, dtype=torch.int32)
    x = rnd(11, 3, 24, dtype=FP, g=g).requires_grad_(True)
    w = rnd(11, 3, 24, dtype=FP, g=g)
    (gx,) = torch.autograd.grad(rope(x, pos, f), x, w)
    check_rope(gx, w, pos, 20, layout, back=True, **kw)
    (gx,) = torch.autograd.grad(rope(x, pos, f).sum(), x)
    check_rope(gx, torch.ones_like(x), pos, 20, layout, back=True, **kw)
    # differences: the map is linear, so only rounding is left; inner products of 792 terms
    d = rnd(11, 3, 24, dtype=FP, g=g)
    (gx,) = torch.autograd.grad(rope(x, pos, f), x, w)
    lhs = float((np64(gx) * np64(d)).sum())
    with torch.no_grad():
        rhs = float(((np64(rope(x + d, pos, f)) - np64(rope(x - d, pos, f))) / 2 * np64(w)).sum())
    size = float((np.abs(np64(w)) * (np.abs(np64(x)) + np.abs(np64(d)))).sum()) * 2 * f.magnitude
    assert abs(lhs - rhs) <= 20 * F * size


def test_rope_second_gradient():
    """The gradient is linear in what comes in: its own gradient is the forward rotation."""
    f = RopeFrequencies(64)
    pos = torch.arange(9, device="cuda")
    x = rnd(9, 2, 64, dtype=FP, g=gen(6)).requires_grad_(True)
    w = rnd(9, 2, 64, dtype=FP, g=gen(7)).requires_grad_(True)
    (gx,) = torch.autograd.grad(rope(x, pos, f), x, w, create_graph=True)
    v = rnd(9, 2, 64, dtype=FP, g=gen(8))
    (gw,) = torch.autograd.grad(gx, w, v)
    check_rope(gw, v, pos, 64, "half")


def test_rope_gradient_in_a_graph():
    """A captured forward and backward pass; refused, with nothing broken, while an eager graph of the same leaf
    is alive (torch itself would break the capture off)."""
    f = RopeFrequencies(64)
    pos = torch.arange(16, device="cuda", dtype=torch.int32)
    x = rnd(16, 2, 64, g=gen(4)).requires_grad_(True)
    w = rnd(16, 2, 64, g=gen(5))
    eager = rope(x, pos, f)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="earlier graph"):
        with torch.cuda.graph(graph):
            rope(x, pos, f)
    torch.randn(3, device="cuda")
    rope(x, pos, f)  # a later graph, gone at once, hides the first from nobody
    with pytest.raises(ValueError, match="earlier graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            rope(x, pos, f)
    (ge,) = torch.autograd.grad(eager, x, w)
    check_rope(ge, w, pos, 64, "half", back=True)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (gx,) = torch.autograd.grad(rope(x, pos, f), x, w)
    graph.replay()
    assert torch.equal(gx, ge)


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------


def make(batch, heads, dim, page, rows, *, dtype=BF, seed=0, spare=2, layout="heads", track=True):
    """A cache whose pages are in no order and hold noise; and its 64-bit twin (rows: capacity asked for)."""
    g = gen(seed)
    each = -(-rows // page)
    pages = batch * each + spare
    if layout == "heads":
        k, v = rnd(pages, heads, page, dim, dtype=dtype, g=g), rnd(pages, heads, page, dim, dtype=dtype, g=g)
    else:  # lines before heads in memory, inside wider rows
        k, v = (rnd(pages, page, heads + 1, dim + 8, dtype=dtype, g=g)[:, :, 1:, 8:].transpose(1, 2) for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[: batch * each]
    c = PagedKVCache(k, v, table.reshape(batch, each).to(torch.int32).cuda(),
                     torch.zeros(2, batch, dtype=torch.int32, device="cuda"),
                     weight=torch.rand(pages, heads, page, device="cuda", generator=g) if track else None,
                     pos=torch.zeros(pages, heads, page, dtype=torch.int32, device="cuda") if track else None)
    return c, twin(c)


def twin(c):
    return Cache(np64(c.k_pages).copy(), np64(c.v_pages).copy(), c.page_table.cpu().numpy(), c.counts.cpu().numpy().copy(),
                 None if c.weight is None else np64(c.weight).copy(), None if c.pos is None else c.pos.cpu().numpy().copy())


def same_rows(c, t, *, k_tol=0.0):
    assert (np.abs(np64(c.k_pages) - t.k) <= k_tol).all()
    assert np.array_equal(np64(c.v_pages), t.v)
    assert np.array_equal(c.counts.cpu().numpy(), t.counts)
    if t.pos is not None:
        assert np.array_equal(c.pos.cpu().numpy(), t.pos)
        assert np.array_equal(np64(c.weight), t.weight, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,page,rotary,layout,pages", [
    (1, 8, 1, 256, 64, 256, "half", "heads"), (5, 4, 2, 128, 16, 64, "interleaved", "lines"),
    (3, 6, 3, 72, 7, 10, "half", "lines"), (2, 3, 3, 8, 1, 2, "interleaved", "heads"),
    (300, 2, 2, 64, 4, 64, "half", "heads"),
])
def test_append(dtype, batch, heads, kv_heads, dim, page, rotary, layout, pages):
    """Ragged prompts with empty ones and padding, then one token of each sequence, then ragged again."""
    g, pygen = gen(7), np.random.default_rng(7)
    f = RopeFrequencies(rotary, layout=layout)
    c, t = make(batch, kv_heads, dim, page, 40, dtype=dtype, layout=pages)
    for step in range(3):
        n = np.ones(batch, dtype=np.int64) if step == 1 else pygen.integers(0, 18, batch)
        if step == 0:
            n[0] = 17
            n[-1] = 0 if batch > 1 else 17
        cu = np.concatenate([[0], np.cumsum(n)])
        total = int(cu[-1]) + (0 if step == 1 else 5)  # 5 of padding
        qkv = rnd(total, heads + 2 * kv_heads, dim, dtype=dtype, g=g)
        q, k, v = qkv[:, :heads], qkv[:, heads : heads + kv_heads], qkv[:, heads + kv_heads :]
        where = np.concatenate([t.counts[1, b] + np.arange(n[b]) for b in range(batch)] + [np.zeros(total - cu[-1])])
        w = torch.rand(total, kv_heads, device="cuda", generator=g) if step == 2 else None
        q_out = torch.full((total, heads, dim), 7.0, dtype=dtype, device="cuda")
        cu_dev = None if step == 1 else torch.tensor(cu, dtype=torch.int32, device="cuda")
        assert c.append(k, v, q=q, freqs=f, cu_tokens=cu_dev, weight=w, q_out=q_out) is q_out
        used = int(cu[-1])
        check_rope(q_out[:used], q[:used], torch.tensor(where[:used]), rotary, layout)
        assert (q_out[used:] == 7).all()
        k_ref, size = rotate(np64(k), where, rotary, layout)
        t.append(k_ref, np64(v), cu, None if w is None else np64(w))
        small = 8 * F * size.max()
        same_rows(c, t, k_tol=small + u(dtype) * (np.abs(t.k) + small) + 2.0**-25)
        t.k = np64(c.k_pages).copy()
    assert c.read_status() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rotary", [0, 2, 4, 8, 12, 20, 40])
@pytest.mark.parametrize("k_skip,v_skip", [(0, 0), (4, 0), (2, 1), (1, 0), (0, 1)])
def test_append_words(layout, rotary, k_skip, v_skip):
    """Every word that pairs, strides and the first row's address allow, for the turned and the copied rows."""
    g, h, d, n = gen(rotary), 3, 40, 13
    c, t = make(1, h, d, 5, 4)
    wide = [rnd(n, h * d + 8, g=g) for _ in range(2)]
    k, v = (w[:, s : s + h * d].unflatten(1, (h, d)) for w, s in zip(wide, (k_skip, v_skip)))
    if rotary == 0:
        c.append(k, v, cu_tokens=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
        t.append(np64(k), np64(v), np.array([0, n]))
        same_rows(c, t)
        return
    q = rnd(n, 2 * d * h + 8, g=g)[:, k_skip : k_skip + 2 * d * h].unflatten(1, (2 * h, d))
    f = RopeFrequencies(rotary, layout=layout)
    out = c.append(k, v, q=q, freqs=f, cu_tokens=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    check_rope(out, q, torch.arange(n), rotary, layout)
    k_ref, size = rotate(np64(k), np.arange(n), rotary, layout)
    t.append(k_ref, np64(v), np.array([0, n]))
    small = 8 * F * size.max()
    same_rows(c, t, k_tol=small + u(BF) * (np.abs(t.k) + small) + 2.0**-25)


def test_append_without_rotation_or_weights():
    c, t = make(2, 2, 64, 16, 30, track=False)
    k, v = rnd(9, 2, 64), rnd(9, 2, 64)
    cu = np.array([0, 4, 9])
    assert c.append(k, v, cu_tokens=torch.tensor(cu, dtype=torch.int32, device="cuda")) is None
    t.append(np64(k), np64(v), cu)
    same_rows(c, t)
    with pytest.raises(ValueError, match="keeps no weights"):
        c.evict(4)
    with pytest.raises(ValueError, match="keeps no weights"):
        c.attend(rnd(2, 2, 64), track=True)


def test_append_beyond_the_pages():
    """Rows with no page are dropped and reported; positions move on, the count stops at the capacity."""
    c, t = make(3, 1, 64, 8, 16)
    c.page_table[1, 1], c.page_table[2, 1] = -1, 99
    t = twin(c)
    k, v = rnd(60, 1, 64), rnd(60, 1, 64)
    cu = np.array([0, 20, 40, 60])
    c.append(k, v, cu_tokens=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    t.append(np64(k), np64(v), cu)
    same_rows(c, t)
    assert c.counts.tolist() == [[16, 16, 16], [20, 20, 20]]
    assert c.read_status() == 0x20 and c.read_status() == 0
    c.append(k[:3], v[:3])
    assert c.counts.tolist() == [[16, 16, 16], [21, 21, 21]] and c.read_status() == 0x20
    t.counts[1] += 1
    same_rows(c, t)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def check_attend(c, t, q, *, valid=None, track=False, scale=None):
    sc = q.shape[2] ** -0.5 if scale is None else scale
    w0 = None if c.weight is None else np64(c.weight).copy()
    out, lse = c.attend(q, key_valid=valid, track=track, scale=scale, return_lse=True)
    v = None if valid is None else valid.cpu().numpy()
    ref, ref_lse, size, reach = t.attend(np64(q), sc, v, track)
    e = (2 * q.shape[2] + 4) * F * reach
    p = 2 * e + 16 * F
    rows = t.counts[0].max()
    tol = u(q.dtype) * np.abs(ref) + (u(q.dtype) + p)[..., None] * (1 + 2**-7) * size
    if q.dtype == HF:  # small probabilities: 2^-25 of the largest each
        tol = tol + rows * 2.0**-25 * np.abs(t.v).max() + 2.0**-25
    err = np.abs(np64(out) - ref)
    assert (err <= tol).all(), (err - tol).max()
    dead = np.isinf(ref_lse)
    assert (np64(out)[dead] == 0).all() and (np64(lse)[dead] == -np.inf).all()
    lse_err = np.abs(np64(lse)[~dead] - ref_lse[~dead])
    assert (lse_err <= (e + 16 * F)[~dead] + 4 * F * np.abs(ref_lse[~dead])).all()
    if track:
        g = q.shape[1] // c.n_kv_heads
        err = np.abs(np64(c.weight) - t.weight)
        assert (err <= F * np.abs(t.weight) + (t.weight - w0) * p.max() + g * F * (t.weight - w0)).all()
        t.weight = np64(c.weight).copy()
    return out


ATTEND = [
    # batch, heads, kv_heads, dim, page, lens, pages
    (1, 8, 1, 256, 64, [1018], "heads"),
    (1, 1, 1, 64, 16, [1], "heads"),
    (6, 4, 2, 128, 16, [0, 1, 15, 64, 65, 700], "lines"),
    (4, 5, 5, 72, 7, [3, 128, 0, 129], "heads"),
    (3, 16, 1, 256, 24, [17, 1, 333], "lines"),
    (2, 40, 2, 128, 8, [100, 63], "heads"),          # 20 query heads of one key-value head: two parts
    (2, 33, 1, 64, 32, [500, 31], "heads"),          # three parts, the last of one head
    (2, 12, 4, 8, 1, [70, 5], "heads"),
    (2, 9, 3, 200, 5, [130, 257], "lines"),
    (1, 4, 1, 128, 64, [9000], "heads"),             # one sequence over every CTA
    (300, 2, 2, 64, 16, [(7 * i) % 50 for i in range(300)], "heads"),
    (2, 2, 1, 96, 100, [20000, 1], "heads"),
    (40, 8, 2, 128, 16, [(53 * i) % 701 for i in range(40)], "heads"),   # 80 pairs: clusters of 2
    (16, 16, 4, 112, 32, [(97 * i) % 900 for i in range(16)], "lines"),  # 64: of 4
    (70, 4, 2, 256, 8, [(31 * i) % 333 for i in range(70)], "heads"),    # 140 of 256 columns: one CTA each
    (160, 2, 1, 256, 8, [(31 * i) % 333 for i in range(160)], "heads"),  # 160: equal shares
    (250, 3, 1, 64, 8, [(31 * i) % 222 for i in range(250)], "heads"),   # 250 of 64: one CTA each
    (330, 9, 3, 64, 16, [(7 * i) % 1000 for i in range(330)], "heads"),  # many of 64 columns: equal shares
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"b{c[0]}h{c[1]}kv{c[2]}d{c[3]}p{c[4]}n{max(c[5])}")
def test_attend(case, masked, dtype):
    batch, heads, kv_heads, dim, page, lens, pages = case
    g = gen(11)
    c, t = make(batch, kv_heads, dim, page, max(max(lens), 1), dtype=dtype, layout=pages)
    c.counts[0] = torch.tensor(lens)
    t.counts[0] = lens
    valid = None
    if masked:  # at random, over a width that ends before some sequences do; the last sequence has none left
        valid = torch.rand(batch, max(max(lens) - 3, 1), device="cuda", generator=g) > 0.3
        if batch > 1:
            valid[-1] = False
    q = rnd(batch, heads + 1, dim, dtype=dtype, g=g, scale=2.0)[:, 1:]
    for track in (False, True):
        out = check_attend(c, t, q, valid=valid, track=track)
        assert torch.equal(c.attend(q, key_valid=valid), out)  # fixed order of every sum
    assert c.read_status() == 0


def test_attend_reads_only_what_counts():
    """NaN and infinities in masked rows, behind the last row, in the heads' gaps and in pages of nobody."""
    c, t = make(3, 2, 64, 16, 100, layout="lines")
    lens = [37, 64, 90]
    c.counts[0] = torch.tensor(lens)
    t.counts[0] = lens
    valid = torch.rand(3, 100, device="cuda", generator=gen(1)) > 0.4
    keep = torch.zeros(c.num_pages, 2, 16, dtype=torch.bool)
    for b in range(3):
        _, p, line = t.rows(b, valid.cpu().numpy())
        keep[p, :, line] = True
    for pages, bad in ((c.k_pages, float("nan")), (c.v_pages, float("inf"))):
        pages.copy_(torch.where(keep.cuda()[..., None], pages, bad))
    check_attend(c, t, rnd(3, 8, 64), valid=valid, track=True)


def test_attend_values_that_are_not_finite():
    """A NaN or infinity in a row that counts reaches the heads that read it, and no other."""
    c, t = make(2, 2, 64, 16, 50)
    c.counts[0] = torch.tensor([40, 50])
    q = rnd(2, 4, 64)
    good = c.attend(q)
    p, line = t.at(0, 33)
    c.v_pages[p, 1, line, 5] = float("inf")
    out = c.attend(q)
    assert torch.isinf(out[0, 2:, 5]).all()
    c.k_pages[p, 1, line, 0] = float("nan")
    out = c.attend(q)
    assert torch.isnan(out[0, 2:]).all()
    assert torch.equal(out[0, :2], good[0, :2]) and torch.equal(out[1], good[1])


def test_attend_large_scores():
    """Scores far apart and far from 0: the running maximum; a scale of 0 (the mean) and a negative one."""
    c, t = make(1, 1, 64, 16, 300)
    c.counts[0] = t.counts[0] = 300
    q = rnd(1, 8, 64, scale=40.0)
    check_attend(c, t, q)
    check_attend(c, t, q, scale=0.0)
    check_attend(c, t, q, scale=-0.3)


def test_attend_two_graphs_at_once():
    """Two captured calls on one cache (read only), replayed on two streams: each has scratch of its own."""
    c, t = make(2, 2, 128, 16, 9000)
    c.counts[0] = torch.tensor([9000, 5000])
    t.counts[0] = [9000, 5000]
    qs = [rnd(2, 8, 128, g=gen(i)) for i in range(2)]
    want = [check_attend(c, t, q) for q in qs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in qs], [], []
    for q, s in zip(qs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(c.attend(q))
        graphs.append(g)
    for _ in range(20):
        for g, s, o in zip(graphs, streams, outs):
            with torch.cuda.stream(s):
                o.zero_()
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want)) and c.read_status() == 0


def test_gradients_are_refused():
    """Nothing that would need one is dropped in silence."""
    c, _ = make(2, 1, 64, 16, 32)
    f, x = RopeFrequencies(64), rnd(2, 1, 64)
    g = x.clone().requires_grad_(True)
    for call in (lambda: c.append(g, x), lambda: c.append(x, g), lambda: c.append(x, x, q=g, freqs=f),
                 lambda: c.attend(g), lambda: rope(g, torch.zeros(2, device="cuda", dtype=torch.int32), f, out=x),
                 lambda: rope(x, torch.zeros(2, device="cuda", dtype=torch.int32), f, out=g)):
        with pytest.raises(ValueError, match="gradient|differentiable"):
            call()
    with torch.no_grad():
        c.append(g, g, q=g, freqs=f)
        c.attend(g)
    assert c.lens.tolist() == [1, 1] and c.read_status() == 0


def test_attend_bad_pages_and_counts():
    c, t = make(3, 1, 64, 16, 64)
    c.page_table[0, 1], c.page_table[0, 2], c.page_table[1, 0] = -7, c.num_pages, 2**31 - 1
    t = twin(c)
    c.counts[0] = torch.tensor([60, 16, 1000])
    t.counts[0] = [60, 16, 1000]
    check_attend(c, t, rnd(3, 2, 64), track=True)
    assert c.read_status() == 0x20
    c.counts[0] = torch.tensor([16, 0, -5])
    t.counts[0] = [16, 0, -5]
    check_attend(c, t, rnd(3, 2, 64), track=True)
    assert c.read_status() == 0x20


def test_attend_shared_pages_two_streams():
    """Two sequences over the same (read-only) pages, and two calls at once on two streams."""
    c, t = make(4, 2, 128, 16, 2000)
    c.page_table[1] = c.page_table[0]
    t = twin(c)
    c.counts[0] = torch.tensor([2000, 1500, 900, 2000])
    t.counts[0] = [2000, 1500, 900, 2000]
    qs = [rnd(4, 8, 128, g=gen(i)) for i in range(2)]
    want = [check_attend(c, t, q) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("batch,heads,dim,page,lens,budget,recent,sinks,pages", [
    (1, 1, 64, 16, [33], 32, 4, 1, "heads"),
    (4, 2, 256, 64, [1, 100, 129, 512], 128, 16, 4, "lines"),
    (3, 3, 72, 7, [50, 0, 31], 1, 1, 0, "heads"),
    (2, 1, 8, 16, [3000, 2100], 700, 0, 0, "heads"),
    (1, 2, 128, 24, [5000], 4999, 2000, 10, "heads"),
    (1, 1, 64, 16, [40], 30, 26, 4, "heads"),        # nothing but protected rows stays
    (40, 4, 64, 16, [(37 * i) % 300 for i in range(40)], 100, 10, 2, "heads"),
    (1, 1, 8, 16, [33000], 20000, 100, 4, "heads"),      # a cluster of CTAs for the one pair
    (1, 2, 8, 16, [20000], 19998, 1000, 4, "lines"),     # two rows to go, in a cluster
    (2, 1, 8, 64, [8200, 30], 8196, 4, 0, "heads"),      # four, in two CTAs
    (1, 1, 8, 16, [8300], 100, 0, 0, "heads"),
    (3, 2, 64, 16, [203, 900, 201], 200, 20, 2, "heads"),  # three to go, one to go, and 700, in pages for many more
])
def test_evict(dtype, batch, heads, dim, page, lens, budget, recent, sinks, pages):
    c, t = make(batch, heads, dim, page, max(lens) + 3, dtype=dtype, layout=pages)
    r = np.random.default_rng(3)
    for b, n in enumerate(lens):
        for i in range(n):
            p, line = t.at(b, i)
            for h in range(heads):
                t.pos[p, h, line] = i if h == 0 else -1
        for h in range(1, heads):  # other heads hold their rows in another order
            order = r.permutation(n)
            for i in range(n):
                p, line = t.at(b, i)
                t.pos[p, h, line] = order[i]
    t.weight[:] = np.float32(r.standard_normal(t.weight.shape))
    coarse = r.random(t.weight.shape) < 0.5  # many ties, zeros of both signs among them
    t.weight[coarse] = np.round(t.weight[coarse] * 2) / 2 * r.choice([1, -1], coarse.sum())
    special = r.random(t.weight.shape)
    for i, v in enumerate((np.nan, np.inf, -np.inf, 1e-42, -1e-42)):
        t.weight[(special > i * 0.01) & (special < (i + 1) * 0.01)] = v
    t.weight = np.float64(np.float32(t.weight))
    t.counts[:] = np.array(lens)
    c.weight.copy_(torch.tensor(t.weight))
    c.pos.copy_(torch.tensor(t.pos))
    c.counts.copy_(torch.tensor(t.counts))
    c.evict(budget, recent=recent, sinks=sinks)
    t.evict(budget, recent, sinks)
    same_rows(c, t)
    c.evict(budget, recent=recent, sinks=sinks)  # nothing is over the budget now
    same_rows(c, t)
    assert c.read_status() == 0


def test_evict_more_rows_than_a_cta_holds():
    """80 sequences, so one CTA each, of up to 50000 rows: keys beyond the shared memory are worked out again."""
    c, t = make(80, 1, 8, 64, 50000, spare=0)
    r = np.random.default_rng(5)
    t.weight[:] = np.float64(np.float32(np.round(r.standard_normal(t.weight.shape), 2)))
    t.pos[:] = r.integers(0, 60000, t.pos.shape)
    t.counts[0, :] = 7
    t.counts[0, [3, 79]] = 50000, 49500
    t.counts[1, :] = 60000
    for x, y in ((c.weight, t.weight), (c.pos, t.pos), (c.counts, t.counts)):
        x.copy_(torch.tensor(y))
    c.evict(20000, recent=500, sinks=4)
    t.evict(20000, 500, 4)
    same_rows(c, t)


def test_strides_of_single_elements():
    """One page, head, line or sequence: whatever stride torch gives that dimension."""
    base = rnd(2, 5, 1, 72)
    k, v = (base[i, :, :, 8:].unsqueeze(1).as_strided((5, 1, 1, 64), (72, 3, 7, 1)) for i in range(2))
    table = torch.tensor([[3]], dtype=torch.int32, device="cuda").as_strided((1, 1), (5, 9))
    c = PagedKVCache(k, v.as_strided((5, 1, 1, 64), (72, 11, 1, 1)), table,
                     torch.tensor([[1], [1]], dtype=torch.int32, device="cuda"))
    t = twin(c)
    valid = torch.ones(1, 1, dtype=torch.bool, device="cuda").as_strided((1, 1), (1, 4))
    check_attend(c, t, rnd(1, 2, 64), valid=valid)
    assert c.read_status() == 0


def test_evict_leaves_a_sequence_with_bad_pages():
    c, t = make(2, 1, 64, 8, 32)
    c.page_table[0, 2] = -1
    c.counts.copy_(torch.tensor([[30, 30], [30, 30]]))
    t = twin(c)
    c.evict(10, recent=2)
    t.evict(10, 2)
    same_rows(c, t)
    assert c.lens.tolist() == [30, 10] and c.read_status() == 0x20
    c.evict(32)  # no sequence can hold more
    assert c.lens.tolist() == [30, 10] and c.read_status() == 0


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def _step(c, f, qkv, budget):
    heads = qkv.shape[1] - 2 * c.n_kv_heads
    q = c.append(qkv[:, heads : heads + c.n_kv_heads], qkv[:, heads + c.n_kv_heads :], q=qkv[:, :heads], freqs=f)
    out = c.attend(q, track=True)
    c.evict(budget, recent=8, sinks=2)
    return q, out


def test_decode_together():
    """Prompts, then decoding at a fixed budget: every step against the 64-bit model, which follows the
    device's own choices (its accumulated weights decide, so a rounding may not send them apart)."""
    batch, heads, kv_heads, dim, budget = 3, 8, 2, 128, 48
    f = RopeFrequencies(dim, scaling="linear", factor=2.0)
    c, t = make(batch, kv_heads, dim, 16, 80)
    g = gen(21)
    n = [70, 5, 44]
    cu = np.concatenate([[0], np.cumsum(n)])
    k, v = rnd(cu[-1], kv_heads, dim, g=g), rnd(cu[-1], kv_heads, dim, g=g)
    w = torch.rand(int(cu[-1]), kv_heads, device="cuda", generator=g)
    c.append(k, v, freqs=f, cu_tokens=torch.tensor(cu, dtype=torch.int32, device="cuda"), weight=w)
    c.evict(budget, recent=8, sinks=2)
    for _ in range(12):
        t = twin(c)
        qkv = rnd(batch, heads + 2 * kv_heads, dim, g=g)
        before = t.counts.copy()
        q = c.append(qkv[:, heads : heads + 2], qkv[:, heads + 2 :], q=qkv[:, :heads], freqs=f)
        check_rope(q, qkv[:, :heads], torch.tensor(before[1]), dim, "half", scaling="linear", factor=2.0)
        t = twin(c)
        assert np.array_equal(t.counts, before + 1)
        check_attend(c, t, q, track=True)
        t = twin(c)
        c.evict(budget, recent=8, sinks=2)
        t.evict(budget, 8, 2)
        same_rows(c, t)
    assert c.lens.tolist() == [48, 17, 48] and c.counts[1].tolist() == [82, 17, 56] and c.read_status() == 0


def test_decode_step_in_a_graph():
    """The captured step replays what the eager one does, on another stream than the cache was made on."""
    budget, f = 40, RopeFrequencies(64)
    c, _ = make(2, 2, 64, 16, 64, seed=5)
    start = torch.tensor([[40, 13], [90, 13]], dtype=torch.int32, device="cuda")
    c.counts.copy_(start)
    c.pos.copy_(torch.randint(0, 90, c.pos.shape, device="cuda", generator=gen(1), dtype=torch.int32))
    keep = [x.clone() for x in (c.k_pages, c.v_pages, c.weight, c.pos)]
    inputs = [rnd(2, 8, 64, g=gen(i)) for i in range(9)]
    want = []
    for x in inputs:
        want.append([y.clone() for y in _step(c, f, x, budget)])
    final = [x.clone() for x in (c.k_pages, c.v_pages, c.weight, c.pos, c.counts)]
    buf = torch.empty_like(inputs[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        _step(c, f, buf.zero_(), budget)
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            q, out = _step(c, f, buf, budget)
        for x, y in zip((c.k_pages, c.v_pages, c.weight, c.pos, c.counts), (*keep, start)):
            x.copy_(y)
        for x, (wq, wo) in zip(inputs, want):
            buf.copy_(x)
            graph.replay()
            assert torch.equal(q, wq) and torch.equal(out, wo)
    s.synchronize()
    for x, y in zip((c.k_pages, c.v_pages, c.weight, c.pos, c.counts), final):
        assert torch.equal(x, y)
    assert c.read_status() == 0


def test_prefix_cache_rows_into_pages():
    """A prefix's dense K/V rows (as the prefix LM leaves them, padded tokens among them) into pages, and a
    token over them: the same as the dense single-token attention."""
    from pi05_infer import abi, ops

    p, heads, dim = 300, 8, 256
    g = gen(31)
    k, v = rnd(1, p, dim, g=g), rnd(1, p, dim, g=g)
    pad = torch.ones(p, dtype=torch.uint8, device="cuda")
    pad[100:140] = 0
    c, t = make(1, 1, dim, 64, 320)
    c.append(k.transpose(0, 1), v.transpose(0, 1), cu_tokens=torch.tensor([0, p], dtype=torch.int32, device="cuda"))
    t = twin(c)
    q = rnd(1, heads, dim, g=g)
    out = check_attend(c, t, q, valid=pad[None])
    dense = torch.empty(heads, dim, dtype=BF, device="cuda")
    abi.attention(q[0], k[0], v[0], pad, dense, dim**-0.5, 0, ops.workspace(q.device))
    # both are within their roundings of the same value: probabilities and output, twice
    size = t.attend(np64(q), dim**-0.5, pad[None].cpu().numpy())[2]
    assert (np.abs(np64(out[0]) - np64(dense)) <= 4.5 * u(BF) * size[0]).all()
