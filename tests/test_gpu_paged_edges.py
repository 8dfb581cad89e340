"""GPU tests of the text-decoding operators at their edges: precision, values that are not finite, overlapping
views, forward-mode derivatives, tables far longer than their sequences.  Model, tolerances and helpers as in
``test_gpu_paged.py``."""

from decimal import localcontext

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from paged_model import turns_of
from test_gpu_paged import BF, F, FP, HF, check_attend, check_rope, gen, make, np64, rnd, same_rows, twin, u

from pi05_infer import PagedKVCache, RopeFrequencies, rope

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# attention: the probabilities' bits
# ---------------------------------------------------------------------------

# batch, heads, kv_heads, dim, rows: a cluster for each pair, then equal shares; up to 8 query heads, then more
BITS = [(2, 8, 1, 256, 900), (3, 8, 2, 80, 500), (2, 12, 1, 128, 700), (2, 8, 2, 128, 20000), (2, 16, 1, 256, 9000),
        (4, 3, 1, 64, 9000)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,rows", BITS)
def test_attend_adds_no_rounding_of_16_bits(dtype, batch, heads, kv_heads, dim, rows):
    """The output is the sum of exact products within fp32's errors and a probability's two 16-bit parts (2^-16 of
    it in bf16, 2^-21 in fp16 and 2^-39 of the largest), rounded once: the last term alone is of the type's size."""
    c, t = make(batch, kv_heads, dim, 64, rows, dtype=dtype)
    t.counts[0] = rows
    c.counts[0] = rows
    q = rnd(batch, heads, dim, dtype=dtype, g=gen(3), scale=2.0)
    out = np64(c.attend(q))
    ref, _, size, reach = t.attend(np64(q), dim**-0.5)
    p = 2 * ((2 * dim + 4) * F * reach) + 16 * F
    parts = 2.0**-16 if dtype == BF else 2.0**-21
    # sums of `rows` products in fp32, in the matrix unit's order: 2 rows 2^-24 at most, and it is far from it
    near = (parts + p)[..., None] * size + 2 * rows * F * size
    if dtype == HF:
        near = near + rows * 2.0**-39 * np.abs(t.v).max() + 2.0**-25
    assert (np.abs(out - ref) <= u(dtype) * (np.abs(ref) + near) + near).all()
    # and so most outputs are the correctly rounded ones
    assert (torch.tensor(ref).to(dtype).double().numpy() == out).mean() > 0.95


@pytest.mark.parametrize("rows,batch", [(1000, 200), (4000, 120)])  # one CTA a pair; equal shares
def test_attend_long_flat_tail(rows, batch):
    """fp16: rows of 2^-25.5 of the largest probability each, which hold all of the values, count."""
    c, t = make(batch, 1, 64, 16, rows, dtype=HF)
    c.k_pages.zero_()
    c.v_pages.fill_(1000.0)
    c.k_pages[..., 0] = -25.5 * np.log(2)
    for b in range(batch):  # the largest in every warp's first tile
        for r in (0, 16, 32, 48):
            p, line = t.at(b, r)
            c.k_pages[p, 0, line, 0] = 0.0
            c.v_pages[p, 0, line] = 0.0
    c.counts[0] = rows
    t = twin(c)
    q = torch.zeros(batch, 2, 64, dtype=HF, device="cuda")
    q[..., 0] = 1.0
    ref, _, size, reach = t.attend(np64(q), 1.0)
    assert ref.min() > 5e-3
    near = (2.0**-21 + 2 * (132 * F * reach) + 16 * F + 2 * rows * F)[..., None] * size + rows * 2.0**-39 * 1000
    assert (np.abs(np64(c.attend(q, scale=1.0)) - ref) <= u(HF) * (ref + near) + near + 2.0**-25).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows", [200, 20000])
def test_attend_infinite_values(dtype, rows):
    """An infinite value of any probability gives that infinity, as a product of whole probabilities does."""
    c, t = make(1, 1, 64, 16, rows, dtype=dtype)
    c.k_pages.zero_()
    weights = [0.0, -1.0, -3.3, -12.0]  # scores of the rows with infinities; 0 for all others
    for i, s in enumerate(weights):
        p, line = t.at(0, 17 * i + 5)
        c.k_pages[p, 0, line, 0] = s
        c.v_pages[p, 0, line, i] = float("inf")
        c.v_pages[p, 0, line, i + 8] = -float("inf")
    c.counts[0] = rows
    q = torch.zeros(1, 3, 64, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    out = c.attend(q, scale=1.0)
    assert (out[..., :4] == float("inf")).all() and (out[..., 8:12] == -float("inf")).all()
    assert torch.isfinite(out[..., 12:]).all() and torch.isfinite(out[..., 4:8]).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows", [150, 20000])  # a cluster for each pair; equal shares, joined
@pytest.mark.parametrize("kv_heads,heads", [(2, 4), (1, 11)])
def test_attend_scores_that_are_not_finite(dtype, rows, kv_heads, heads):
    """Rows that count and score -inf, all of them: softmax is 0 / 0, NaN, for the output and their weights, and
    log 0 for the sum; some of them: nothing.  Masked rows add nothing to their weight whatever the others hold."""
    g = gen(5)
    c, t = make(4, kv_heads, 64, 16, rows, dtype=dtype)
    c.k_pages.copy_(c.k_pages.abs())
    q = rnd(4, heads, 64, dtype=dtype, g=g).abs() + 0.1
    valid = torch.rand(4, rows, device="cuda", generator=g) > 0.3
    valid[1] = False
    c.counts[0] = rows
    good, good_lse = c.attend(q, key_valid=valid, return_lse=True)
    live = valid.cpu().numpy()
    spoiled = np.zeros((4, rows), dtype=bool)
    spoiled[0] = spoiled[1] = True       # all; all, but masked
    spoiled[2] = ~live[2]                # masked rows alone: the result stays
    bad = np.flatnonzero(live[3])[:1]    # one NaN
    at = torch.arange(rows, device="cuda")
    for b in range(4):
        r = at[torch.tensor(spoiled[b], device="cuda")]
        c.k_pages[c.page_table[b, r // 16].long(), :, r % 16, 3] = -float("inf")
    p, line = t.at(3, int(bad[0]))
    c.k_pages[p, :, line, 0] = float("nan")
    before = c.weight.clone()
    out, lse = c.attend(q, key_valid=valid, return_lse=True, track=True)
    assert torch.isnan(out[0]).all() and (lse[0] == -float("inf")).all()
    assert (out[1] == 0).all() and (lse[1] == -float("inf")).all()
    assert torch.equal(out[2], good[2]) and torch.equal(lse[2], good_lse[2])
    assert torch.isnan(out[3]).all() and torch.isnan(lse[3]).all()
    for b in range(4):
        pg, line = c.page_table[b, at // 16].long(), at % 16
        was, now = before[pg, :, line], c.weight[pg, :, line]
        assert torch.equal(was[~valid[b]], now[~valid[b]])
        counted = now[valid[b]]
        assert torch.isnan(counted).all() if b in (0, 3) else torch.isfinite(counted).all()
    c.k_pages[p, :, line[int(bad[0])], 0] = 0  # and one row of -inf among others is left out
    p2, line2 = t.at(3, int(bad[0]))
    c.k_pages[p2, :, line2, 0], c.k_pages[p2, :, line2, 1] = 0, -float("inf")
    without = valid.clone()
    without[3, int(bad[0])] = False
    assert torch.equal(c.attend(q, key_valid=valid)[3], c.attend(q, key_valid=without)[3])


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


def overlapping():
    g = gen(8)
    return [
        rnd(6, 66, g=g).unfold(1, 64, 1),                                  # heads one value apart
        rnd(73, g=g).unfold(0, 64, 1).unsqueeze(1),                        # tokens one value apart
        rnd(1, 3, 64, g=g).expand(5, 3, 64), rnd(5, 1, 64, g=g).expand(5, 3, 64),
        rnd(200, g=g).as_strided((4, 5, 64), (16, 8, 1)),
    ]


@pytest.mark.parametrize("case", range(5))
def test_rope_of_overlapping_views(case):
    """The same as of a copy, forward and for such a view as the incoming gradient."""
    x = overlapping()[case]
    f, pos = RopeFrequencies(64), torch.arange(x.shape[0], device="cuda") * 7
    want = rope(x.contiguous(), pos, f)
    check_rope(want, x, pos, 64, "half")
    assert torch.equal(rope(x, pos, f), want)
    leaf = x.contiguous().requires_grad_(True)
    (gx,) = torch.autograd.grad(rope(leaf, pos, f), leaf, x)
    assert torch.equal(gx, rope(x.contiguous(), pos, f, transpose=True))
    leaf = x.detach().requires_grad_(True)  # an overlapping leaf
    (gx,) = torch.autograd.grad(rope(leaf, pos, f), leaf, torch.ones_like(want))
    assert torch.equal(gx, rope(torch.ones_like(want), pos, f, transpose=True))


def test_rope_into_overlapping_views_is_refused():
    x = rnd(6, 3, 64)
    f, pos = RopeFrequencies(64), torch.arange(6, device="cuda")
    for out in (rnd(6, 66).unfold(1, 64, 1), rnd(1, 3, 64).expand(6, 3, 64), rnd(6, 1, 64).expand(6, 3, 64),
                rnd(700).as_strided((6, 3, 64), (64, 64, 1)), rnd(700).as_strided((6, 3, 64), (100, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            rope(x, pos, f, out=out)
    want = rope(x, pos, f)
    for out in (rnd(3, 6, 70)[:, :, 3:67].transpose(0, 1), rnd(6, 4, 64)[:, 1:], rnd(6, 3, 64)):
        assert torch.equal(rope(x, pos, f, out=out), want)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("reverse", [False, True])
def test_rope_forward_mode(layout, reverse):
    """The tangent turns as the values do (the map is linear), whether or not a gradient is wanted as well."""
    f, pos = RopeFrequencies(20, layout=layout), torch.arange(7, device="cuda") * 11
    x, d = rnd(7, 3, 24, g=gen(1)).requires_grad_(reverse), rnd(7, 24, 3, g=gen(2)).transpose(1, 2)
    want, turned = rope(x.detach(), pos, f), rope(d.contiguous(), pos, f)
    with forward_ad.dual_level():
        y = rope(forward_ad.make_dual(x, d), pos, f)
        value, tangent = forward_ad.unpack_dual(y)
        assert torch.equal(value, want) and torch.equal(tangent, turned)
        if reverse:
            w = torch.ones_like(want)
            assert torch.equal(torch.autograd.grad(value, x, w)[0], rope(w, pos, f, transpose=True))
    with torch.no_grad(), forward_ad.dual_level():
        assert torch.equal(forward_ad.unpack_dual(rope(forward_ad.make_dual(x, d), pos, f, transpose=True)).tangent,
                           rope(d.contiguous(), pos, f, transpose=True))


def test_forward_mode_is_refused_where_it_would_be_lost():
    c, _ = make(2, 1, 64, 16, 32)
    f, pos, x, t = RopeFrequencies(64), torch.arange(2, device="cuda"), rnd(2, 1, 64), rnd(2, 1, 64)
    with forward_ad.dual_level():
        g = forward_ad.make_dual(x.clone(), t)
        for call in (lambda: c.append(g, x), lambda: c.append(x, g), lambda: c.append(x, x, q=g, freqs=f),
                     lambda: c.attend(g), lambda: rope(g, pos, f, out=x), lambda: rope(x, pos, f, out=g)):
            with pytest.raises(ValueError, match="gradient|differentiable"):
                call()
        c.append(x, x, q=x, freqs=f)  # within a level, but without tangents
        c.attend(x)
        rope(x, pos, f, out=x)
    assert c.lens.tolist() == [1, 1] and c.read_status() == 0


def test_recording_is_refused():
    """torch.jit.trace and make_fx see no call of the library: what they recorded would return unwritten memory.
    torch.compile leaves the calls to Python, and modes that only look on change nothing."""
    f, pos = RopeFrequencies(64), torch.arange(3, device="cuda")
    c, _ = make(3, 2, 64, 16, 32)
    x, y = rnd(3, 2, 64, g=gen(1)), rnd(3, 2, 64, g=gen(2))

    def step(k):
        c.append(k, k)
        return c.attend(k)

    def evict(k):
        c.evict(8)
        return k + 1

    for call in (lambda k: rope(k, pos, f), lambda k: rope(k, pos, f, out=k), step, lambda k: c.attend(k), evict):
        for record in (lambda: torch.jit.trace(call, (x,), check_trace=False), lambda: make_fx(call)(x),
                       lambda: make_fx(call, pre_dispatch=True)(x)):
            with pytest.raises(ValueError, match="cannot be recorded"):
                record()
    assert c.lens.tolist() == [0, 0, 0] and c.read_status() == 0
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(ValueError, match="cannot be recorded"):
        make_fx(lambda k: torch.autograd.grad(rope(k, pos, f), k, y)[0])(leaf)
    compiled, whole = torch.compile(lambda k: rope(k, pos, f) * 2, backend="eager"), torch.compile(step, backend="eager")
    for k in (x, y, x):
        assert torch.equal(compiled(k), rope(k, pos, f) * 2)
        c.counts.zero_()
        want = step(k)
        c.counts.zero_()
        assert torch.equal(whole(k), want) and c.lens.tolist() == [1, 1, 1]
    with FlopCounterMode(display=False):
        assert torch.equal(rope(x, pos, f), rope(x, pos, f))


def test_writes_are_seen_by_autograd():
    """A tensor that a graph saved and a call then wrote to: the backward pass is refused."""
    c, _ = make(2, 1, 64, 16, 32)
    f, pos, x = RopeFrequencies(64), torch.arange(2, device="cuda"), rnd(2, 1, 64)
    c.append(x, x)
    y, z = torch.empty_like(x), torch.empty_like(x)
    state = dict(k=c.k_pages, v=c.v_pages, weight=c.weight)
    for call, names in ((lambda: c.append(x, x, q=x, freqs=f, q_out=y), ("k", "v", "weight", "y")),
                        (lambda: c.attend(x, track=True), ("weight",)), (lambda: c.attend(x, out=y), ("y",)),
                        (lambda: c.evict(1), ("k", "v", "weight")), (lambda: rope(x, pos, f, out=y), ("y",))):
        for name, t in (*state.items(), ("y", y), ("z", z)):
            w = torch.ones((), device="cuda", dtype=t.dtype, requires_grad=True)
            loss = (t * w).sum()
            before = c.counts._version
            call()
            assert (c.counts._version > before) == ("k" in names)
            if name in names:
                with pytest.raises(RuntimeError, match="inplace operation"):
                    loss.backward()
            else:
                loss.backward()
    with torch.inference_mode():
        out = rnd(2, 1, 64)
        rope(x, pos, f, out=out)
        c.append(x, x, q=x, freqs=f, q_out=out)
    rope(x, pos, f, out=out)  # made in inference mode, without a version


@pytest.mark.parametrize("forward", [False, True])
def test_gradients_of_what_is_written_are_refused(forward):
    """Outputs given by the caller, new weights and the cache's own tensors: in reverse and in forward mode."""
    f, x = RopeFrequencies(64), rnd(2, 1, 64)

    def wanting(t):
        return forward_ad.make_dual(t.clone(), torch.ones_like(t)) if forward else t.clone().requires_grad_(True)

    with forward_ad.dual_level():
        c, _ = make(2, 1, 64, 16, 32)
        o, w = wanting(x), wanting(torch.ones(2, 1, device="cuda"))
        calls = [lambda: c.append(x, x, q=x, freqs=f, q_out=o), lambda: c.append(x, x, weight=w), lambda: c.attend(x, out=o)]
        for name in ("k", "v", "weight"):
            t = dict(k=c.k_pages, v=c.v_pages, weight=c.weight)
            t[name] = wanting(t[name])
            d = PagedKVCache(t["k"], t["v"], c.page_table, c.counts, weight=t["weight"], pos=c.pos)
            calls += [lambda d=d: d.append(x, x), lambda d=d: d.attend(x, track=True), lambda d=d: d.evict(1)]
        for call in calls:
            with pytest.raises(ValueError, match="not differentiable"):
                call()
        assert c.lens.tolist() == [0, 0]
        d.attend(x)  # has nothing to do with the weights
        if not forward:
            with torch.no_grad():
                for call in calls:
                    call()
    assert c.read_status() == 0


@pytest.mark.parametrize("budget,recent,sinks", [(2**32 + 8, 0, 0), (2**33 + 8, 2**32 + 2, 1), (2**63, 2**62, 2**62),
                                                 (32, 0, 0), (33, 1, 32)])
def test_evict_numbers_beyond_32_bits(budget, recent, sinks):
    """A budget that no sequence can reach leaves everything as it is, however large the number."""
    c, t = make(2, 1, 64, 16, 32)
    c.counts.fill_(30)
    t = twin(c)
    c.evict(budget, recent=recent, sinks=sinks)
    same_rows(c, t)
    assert c.read_status() == 0


def test_caches_that_the_library_does_not_take():
    """Refused when they are made, not by the first call; and before the workspace is allocated."""
    def build(pages=4, heads=1, page=16, dim=64, batch=2, each=2, skip=0, wide=0, counts=None):
        k = torch.zeros(pages * heads * page * (dim + wide) + skip, dtype=BF, device="cuda")[skip:]
        k = k.view(pages, heads, page, dim + wide)[..., :dim]
        table = torch.zeros(batch, each, dtype=torch.int32, device="cuda")
        counts = torch.zeros(2 * batch, dtype=torch.int32, device="cuda") if counts is None else counts
        return PagedKVCache(k, k, table, counts.view(2, batch))

    build()
    build(skip=8, wide=8)
    for kw in (dict(dim=60), dict(dim=264), dict(skip=4), dict(wide=4), dict(pages=0), dict(heads=0), dict(page=0),
               dict(batch=0), dict(each=0)):
        with pytest.raises(ValueError, match="not a cache that the library takes"):
            build(**kw)
    k = torch.zeros(1, 1, 1 << 20, 8, dtype=BF, device="cuda")
    before = torch.cuda.memory_allocated()
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(1, 2048).contiguous()
    with pytest.raises(ValueError, match="bad cache shape"):  # 2^31 rows
        PagedKVCache(k, k, table, torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    assert torch.cuda.memory_allocated() - before < 1 << 20


def test_rows_with_strides_of_single_elements():
    """One token or one head: whatever stride torch has for it, beyond 31 bits too, and in place with two kinds."""
    f, pos = RopeFrequencies(64), torch.tensor([5], device="cuda")
    far = 2**31 + 5
    x = rnd(1, 3, 64)
    odd = x.as_strided((1, 3, 64), (far, 64, 1))
    want = rope(x, pos, f)
    assert torch.equal(rope(odd, pos, f), want)
    assert torch.equal(rope(x, pos, f, out=torch.empty_like(x).as_strided((1, 3, 64), (1, 64, 1))), want)
    in_place = x.clone()
    rope(in_place.as_strided((1, 3, 64), (far, 64, 1)), pos, f, out=in_place)
    assert torch.equal(in_place, want)
    heads = rnd(4, 1, 64)
    four = torch.arange(4, device="cuda")
    assert torch.equal(rope(heads.as_strided((4, 1, 64), (64, far, 1)), four, f), rope(heads, four, f))
    c, t = make(1, 1, 64, 16, 32)
    k, v, q = rnd(1, 1, 64), rnd(1, 1, 64), rnd(1, 1, 64)
    views = [y.as_strided((1, 1, 64), (far, far + 1, 1)) for y in (k, v, q)]
    c.counts.zero_()
    a = c.append(views[0], views[1], q=views[2], freqs=f), c.k_pages.clone(), c.v_pages.clone()
    c.counts.zero_()
    b = c.append(k, v, q=q, freqs=f), c.k_pages, c.v_pages
    assert all(torch.equal(y, z) for y, z in zip(a, b)) and c.read_status() == 0


def test_rope_of_no_heads():
    f, pos = RopeFrequencies(64), torch.arange(5, device="cuda")
    x = torch.empty(5, 0, 64, dtype=BF, device="cuda")
    assert rope(x, pos, f).shape == (5, 0, 64) and rope(x, pos, f, out=x) is x
    leaf = x.clone().requires_grad_(True)
    assert torch.autograd.grad(rope(leaf, pos, f), leaf, x)[0].shape == (5, 0, 64)


@pytest.mark.parametrize("kw", [
    dict(), dict(scaling="linear", factor=3.0), dict(scaling="ntk", factor=8.0, base=500000.0),
    dict(scaling="yarn", factor=16.0, original=8192),
])
def test_rope_angles_of_far_positions(kw):
    """(1, 0) turns to cos and sin: within 4 fp32 roundings of the exact ones, 2 each for the functions, 1.5 for the
    angle's 2^-28 turn beyond a quarter and half a one for the table's 2^-65 turn a position up to 2^36, more beyond."""
    f = RopeFrequencies(64, layout="interleaved", **{("original_len" if k == "original" else k): v for k, v in kw.items()})
    g = np.random.default_rng(3)
    pos = [0, 1, -1, 2, 12345, 10**6 + 1, 10**9, 2**31 - 1, -(2**31), 2**40 + 3, -(2**45) - 1]
    pos += g.integers(-(2**36), 2**36, 400).tolist() + g.integers(-(2**31), 2**31, 400).tolist()
    x = torch.zeros(len(pos), 1, 64, dtype=FP, device="cuda")
    x[..., 0::2] = 1.0
    y = np64(rope(x, torch.tensor(pos, device="cuda"), f))[:, 0]
    with localcontext() as context:
        context.prec = 50
        turn = np.array([[float(n * t - round(n * t)) for t in turns_of(64, **kw)] for n in pos])
    far = np.abs(np.array(pos, dtype=np.float64))[:, None] * 2.0**-65 * 2 * np.pi
    tol = (4 * F + np.maximum(far - F, 0)) * f.magnitude + F * f.magnitude  # and the product with the magnitude
    assert (np.abs(y[:, 0::2] - np.cos(2 * np.pi * turn) * f.magnitude) <= tol).all()
    assert (np.abs(y[:, 1::2] - np.sin(2 * np.pi * turn) * f.magnitude) <= tol).all()


# ---------------------------------------------------------------------------
# tables far longer than their sequences
# ---------------------------------------------------------------------------


def long_table(batch, heads, dim, page, lens, each, *, dtype=BF, seed=0):
    """A pool for `lens` rows a sequence, behind a table of `each` pages a sequence, no page in the rest of it."""
    c, _ = make(batch, heads, dim, page, max(lens), dtype=dtype, seed=seed)
    table = torch.full((batch, each), -1, dtype=torch.int32, device="cuda")
    table[:, : c.pages_per_seq] = c.page_table
    d = PagedKVCache(c.k_pages, c.v_pages, table, c.counts, weight=c.weight, pos=c.pos)
    d.counts[:] = torch.tensor(lens)
    return d, twin(d)


@pytest.mark.parametrize("budget", [100, 40, 198])  # moved by a kernel of their own, on the spot, a few rows
def test_evict_behind_a_long_table(budget):
    """The workspace goes by the pool where the table reaches further; what is evicted does not change."""
    lens = [200 - 7 * (i % 9) for i in range(40)]
    c, t = long_table(40, 2, 64, 16, lens, 4096)
    assert c.workspace.numel() < (1 << 16) + c.num_pages * 2 * 16 * 4
    r = np.random.default_rng(2)
    t.pos[:] = r.integers(0, 200, t.pos.shape)
    t.weight[:] = np.round(r.standard_normal(t.weight.shape), 1).astype(np.float32)
    c.pos.copy_(torch.tensor(t.pos))
    c.weight.copy_(torch.tensor(t.weight))
    for left in (budget, budget // 2):
        c.evict(left, recent=10, sinks=2)
        t.evict(left, 10, 2)
        same_rows(c, t)
    assert c.read_status() == 0


def test_workspace_of_a_cache_without_weights():
    c = PagedKVCache.allocate(8, 16, 2, 64, 64, 8192, track=False)
    assert c.workspace.numel() <= 1 << 15
    c.page_table[:, 0] = 3
    c.counts[0] = 5
    assert c.attend(rnd(64, 2, 64)).shape == (64, 2, 64) and c.read_status() == 0


@pytest.mark.parametrize("batch,heads,kv_heads", [(160, 8, 2), (100, 18, 1)])
def test_attend_behind_a_long_table(batch, heads, kv_heads):
    """Tracked: the scratch goes by the pool where the table reaches further; what is computed does not change."""
    lens = [1 + (37 * i) % 300 for i in range(batch)]
    lens[0] = 0
    c, t = long_table(batch, kv_heads, 64, 16, lens, 8192)
    valid = torch.rand(batch, 250, device="cuda", generator=gen(4)) > 0.2
    need = c._need(heads, True)[0] - c._need(heads, False)[0]
    assert need < (64 << 20) + (1 << 16) + batch * heads * 64
    check_attend(c, t, rnd(batch, heads, 64, g=gen(1)), valid=valid, track=True)
    assert c.read_status() == 0


def test_attend_tracks_no_more_rows_than_the_pool_has():
    """Pages that stand in several sequences (not allowed to a call that writes), so many that the scores have no
    room: the weights stay, the status says so, and the output is that of a call that only reads."""
    k, v = rnd(4, 1, 16, 64), rnd(4, 1, 16, 64)
    weight = torch.rand(4, 1, 16, device="cuda")
    table = torch.zeros(96, 8192, dtype=torch.int32, device="cuda")
    counts = torch.full((2, 96), 16 * 8192, dtype=torch.int32, device="cuda")
    c = PagedKVCache(k, v, table, counts, weight=weight, pos=torch.zeros(4, 1, 16, dtype=torch.int32, device="cuda"))
    q, before = rnd(96, 2, 64), weight.clone()
    want = c.attend(q)
    assert c.read_status() == 0
    assert torch.equal(c.attend(q, track=True), want) and torch.equal(weight, before)
    assert c.read_status() == 0x20


# ---------------------------------------------------------------------------
# every kernel that the sizes choose
# ---------------------------------------------------------------------------

# batch, heads, kv_heads, dim, page, lens, pages a sequence that the table has room for
KERNELS = [
    # heads of 129 to 160 and of 161 to 192 columns: a cluster for each pair, then equal shares
    (3, 4, 2, 136, 16, [0, 77, 300], 20), (3, 4, 2, 160, 16, [1, 130, 300], 20), (2, 3, 1, 176, 8, [65, 200], 30),
    (2, 8, 1, 192, 24, [500, 3], 30),
    (3, 4, 2, 136, 16, [0, 77, 900], 4096), (3, 4, 2, 160, 16, [1, 130, 900], 4096), (2, 3, 1, 176, 8, [65, 700], 4096),
    (2, 8, 1, 192, 24, [1500, 3], 4096),
    # 9 to 16 query heads of a key-value head: clusters, then equal shares
    (2, 9, 1, 72, 16, [40, 333], 30), (2, 32, 2, 96, 16, [63, 200], 20), (2, 10, 1, 160, 16, [129, 64], 20),
    (1, 16, 1, 192, 16, [250], 16),
    (2, 9, 1, 72, 16, [40, 900], 4096), (2, 32, 2, 96, 16, [63, 700], 4096), (2, 10, 1, 160, 16, [129, 1000], 4096),
    (2, 16, 1, 192, 16, [250, 1], 4096), (3, 30, 2, 256, 16, [700, 0, 65], 4096), (2, 12, 1, 200, 16, [128, 129], 4096),
    (2, 13, 1, 64, 16, [900, 1], 4096), (2, 16, 1, 128, 16, [2000, 17], 4096),
    # more than 16, in parts
    (2, 17, 1, 72, 16, [40, 500], 64), (2, 34, 2, 96, 16, [63, 300], 64), (2, 33, 1, 160, 16, [129, 400], 64),
    (1, 20, 1, 192, 16, [700], 64), (2, 48, 2, 256, 16, [1, 600], 64), (1, 24, 1, 128, 8, [3000], 400),
    # one long sequence among many pairs: more chunks of it to track than CTAs that do
    (256, 2, 1, 64, 16, [9001] + [3] * 255, 600), (130, 18, 2, 64, 16, [4300] + [(5 * i) % 9 for i in range(129)], 300),
]


def pooled(batch, heads, dim, page, lens, each, *, dtype=BF, seed=0):
    """A cache with just the pages that `lens` rows take, in no order, behind a table of `each` pages a sequence."""
    g = gen(seed)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 1
    k, v = (rnd(pages, heads, page, dim, dtype=dtype, g=g) for _ in range(2))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((batch, each), -1, dtype=torch.int32)
    for b, n in enumerate(used):
        table[b, :n] = order[sum(used[:b]) : sum(used[:b]) + n]
    c = PagedKVCache(k, v, table.cuda(), torch.tensor([lens, lens], dtype=torch.int32, device="cuda"),
                     weight=torch.rand(pages, heads, page, device="cuda", generator=g),
                     pos=torch.zeros(pages, heads, page, dtype=torch.int32, device="cuda"))
    return c, twin(c)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", KERNELS, ids=lambda c: f"b{c[0]}h{c[1]}kv{c[2]}d{c[3]}n{max(c[5])}t{c[6]}")
def test_attend_every_kernel(case, dtype):
    batch, heads, kv_heads, dim, page, lens, each = case
    c, t = pooled(batch, kv_heads, dim, page, lens, each, dtype=dtype)
    g = gen(13)
    q = rnd(batch, heads, dim, dtype=dtype, g=g, scale=2.0)
    valid = torch.rand(batch, max(max(lens) - 2, 1), device="cuda", generator=g) > 0.3
    check_attend(c, t, q)
    check_attend(c, t, q, valid=valid, track=True)
    assert c.read_status() == 0


# ---------------------------------------------------------------------------
# padding and eviction
# ---------------------------------------------------------------------------


def test_padded_prompts_and_eviction():
    """Left-padded prompts for a cache that evicts: their tokens alone are appended, and attended to without a mask;
    until an eviction that is the same as all of them under the mask."""
    batch, n, heads, dim, f = 3, 90, 8, 64, RopeFrequencies(64)
    pad = [0, 25, 60]
    g = gen(9)
    k, v, q = rnd(batch, n, 2, dim, g=g), rnd(batch, n, 2, dim, g=g), rnd(batch, heads, dim, g=g)
    valid = torch.arange(n, device="cuda")[None] >= torch.tensor(pad, device="cuda")[:, None]
    padded, _ = make(batch, 2, dim, 16, 100)
    padded.append(k.flatten(0, 1), v.flatten(0, 1), cu_tokens=torch.arange(4, dtype=torch.int32, device="cuda") * n)
    c, _ = make(batch, 2, dim, 16, 100)
    cu = torch.tensor(np.concatenate([[0], np.cumsum([n - p for p in pad])]), dtype=torch.int32, device="cuda")
    c.append(k[valid], v[valid], cu_tokens=cu)
    both = padded.attend(q, key_valid=valid), check_attend(c, twin(c), q, track=True)
    # the same sums in another order, each output within its own tolerance: two roundings, and fp32's
    assert (np.abs(np64(both[0]) - np64(both[1])) <= 2 * u(BF) * np.abs(np64(both[1])) + 2.0**-12).all()
    for step in range(3):
        t = twin(c)
        c.evict(40 - 5 * step, recent=8, sinks=2)
        t.evict(40 - 5 * step, 8, 2)
        same_rows(c, t)
        check_attend(c, t, q, track=True)
        q = c.append(rnd(batch, 2, dim, g=g), rnd(batch, 2, dim, g=g), q=q, freqs=f)
    assert c.read_status() == 0
