"""Cases of the text-decoding operators: rotary positions, the paged key-value cache's append, its single-token
attention and its eviction by accumulated attention weight.

Each case is one call as a serving (or fine-tuning) program makes it.  ``run`` computes it in a plain form with
elementary torch operations, or, where ``own`` is true, with this package's kernels.  A cache is

  k_pages, v_pages  [num_pages, kv_heads, page, dim]   rows of the tokens, keys already rotated
  weight, pos       [num_pages, kv_heads, page]        accumulated attention weight (fp32), position (int32) of a row
  page_table        [batch, pages of a sequence] int32
  counts            [2, batch] int32                   rows in the cache, and tokens seen so far, of each sequence
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pi05-infer_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import pi05_infer

    return pi05_infer


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    half = dict(layout="half", scaling="none", factor=1.0, original=0, base=10000.0)
    return [
        # one token's q|k heads of the 8 + 1 head decoder, in the q|k|v row: the smallest call, all latency
        dict(name="rope-token", op="rope", tokens=1, heads=9, extra=1, dim=256, rotary=256, dtype="bf16", max_pos=1018,
             grad=False, **half),
        # the 968-token prefix of three camera views and a prompt
        dict(name="rope-prefix", op="rope", tokens=968, heads=9, extra=1, dim=256, rotary=256, dtype="bf16",
             max_pos=968, grad=False, **half),
        # fine-tuning on long packed sequences: forward and gradient, half of each head rotated, scaled 16x
        dict(name="rope-long-grad", op="rope", tokens=32768, heads=32, extra=0, dim=128, rotary=64, dtype="bf16",
             max_pos=131072, grad=True, layout="interleaved", scaling="yarn", factor=16.0, original=8192,
             base=10000.0),
        # one new token of each of 64 sequences: rotate q and k, write k and v behind each sequence's last row
        dict(name="append-token", op="append", batch=64, tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, page=16,
             dtype="bf16", seen=2000, one=True, **half),
        # eight ragged prompts into fresh pages
        dict(name="append-prompts", op="append", batch=8, tokens=16384, heads=8, kv_heads=1, dim=256, rotary=256,
             page=64, dtype="bf16", seen=0, one=False, **half),
        # one new token over a 968-token prefix and 50 rows more, padded rows masked: latency
        dict(name="attend-prefix", op="attend", batch=1, heads=8, kv_heads=1, dim=256, page=64, dtype="bf16",
             shortest=1018, longest=1018, masked=True, track=False),
        # a serving batch of 64 sequences of very different lengths, weights accumulated for a later eviction
        dict(name="attend-batch", op="attend", batch=64, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16",
             shortest=17, longest=8192, masked=False, track=True),
        # two long contexts: the work has to be split over the length
        dict(name="attend-long", op="attend", batch=2, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16",
             shortest=131072, longest=131072, masked=False, track=False),
        # a key-value head for each query head, an odd page, fp16, short and ragged
        dict(name="attend-heads", op="attend", batch=24, heads=16, kv_heads=16, dim=80, page=24, dtype="fp16",
             shortest=1, longest=1500, masked=True, track=True),
        # decoding at a fixed budget: each of 64 sequences appends a token and gives up one row of each head
        dict(name="evict-token", op="evict", batch=64, tokens=64, kv_heads=8, dim=128, page=16, dtype="bf16",
             budget=2048, recent=256, sinks=4, one=True),
        # eight ragged prompts cut down to the budget after their prefill
        dict(name="evict-prompts", op="evict", batch=8, tokens=16384, kv_heads=1, dim=256, page=64, dtype="bf16",
             budget=1024, recent=128, sinks=4, one=False),
        # one long prompt cut down to an eighth
        dict(name="evict-long", op="evict", batch=1, tokens=65536, kv_heads=8, dim=128, page=64, dtype="bf16",
             budget=8192, recent=512, sinks=4, one=False),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _draw_rope(rng, dim):
    rotary = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
    scaling = rng.choice(["none", "none", "linear", "ntk", "yarn"])
    if rotary < 4:
        scaling = "none"
    return dict(rotary=rotary, layout=rng.choice(["half", "interleaved"]), scaling=scaling,
                factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
                original=8192 if scaling == "yarn" else 0, base=rng.choice([10000.0, 500000.0]))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "evict", "evict"])
    dim = rng.choice([64, 72, 80, 96, 128, 128, 160, 256, 256])
    page = rng.choice([8, 16, 16, 24, 32, 64, 64, 100, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 1, 2, 4, 8, 16])
    if op == "rope":
        heads = rng.choice([1, 2, 5, 8, 9, 16, 32, 40])
        tokens = _spread(rng, 1, 32768 * 32 * 128 // (heads * dim))
        tokens = min(tokens, 100000)
        return dict(op="rope", tokens=tokens, heads=heads, extra=rng.choice([0, 0, 1]), dim=dim,
                    dtype=rng.choice([dtype, dtype, "fp32"]) if tokens * heads * dim < 1 << 26 else dtype,
                    max_pos=max(tokens, _spread(rng, 1, 4000000)), grad=rng.random() < 0.5, **_draw_rope(rng, dim))
    if op == "append":
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        one = rng.random() < 0.4
        batch = _spread(rng, 1, 256) if one else _spread(rng, 1, 24)
        most = 16384 * 10 * 256 // ((heads + 2 * kv_heads) * dim)
        tokens = batch if one else max(batch, _spread(rng, 1, most))
        return dict(op="append", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    dtype=dtype, seen=_spread(rng, 1, 2000) - 1 if one else 0, one=one, **_draw_rope(rng, dim))
    if op == "attend":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
        batch = _spread(rng, 1, 128)
        most = max(1, min(131072, (1 << 28) // (batch * kv_heads * dim)))
        longest = _spread(rng, 1, most)
        shortest = longest if rng.random() < 0.3 else min(longest, _spread(rng, 1, longest))
        return dict(op="attend", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                    shortest=shortest, longest=longest, masked=rng.random() < 0.4, track=rng.random() < 0.5)
    one = rng.random() < 0.5
    batch = _spread(rng, 1, 64) if one else _spread(rng, 1, 12)
    most = max(64, min(65536 if not one else 8192, (1 << 26) // (kv_heads * dim * (batch if one else 1))))
    budget = _spread(rng, 16, most if one else max(16, most // 4))
    tokens = batch if one else max(batch, _spread(rng, budget, most))
    sinks = rng.choice([0, 1, 4])
    return dict(op="evict", batch=batch, tokens=tokens, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                budget=budget, recent=rng.randint(1, max(1, (budget - sinks) // 2)), sinks=sinks, one=one)


def _lengths(case):
    """The cache lengths of an attend case, evenly spread between the shortest and the longest."""
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def work(case):
    op, es = case["op"], 4 if case["dtype"] == "fp32" else 2
    d = case["dim"]
    if op == "rope":
        n = case["tokens"] * case["heads"] * d
        k = 2 if case["grad"] else 1
        return {"bytes": k * (2 * n * es + 4 * case["tokens"]),
                "flops": k * 3 * case["tokens"] * case["heads"] * case["rotary"]}
    if op == "attend":
        rows = sum(_lengths(case)) * case["kv_heads"]
        b = rows * d * 2 * es + 2 * case["batch"] * case["heads"] * d * es + 4 * case["batch"] * case["heads"]
        b += sum(_lengths(case)) if case["masked"] else 0
        return {"bytes": b + (8 * rows if case["track"] else 0),
                "flops": 4 * sum(_lengths(case)) * case["heads"] * d}
    rows = case["tokens"] * case["kv_heads"]
    move = rows * (4 * d * es + 8)  # k and v read and written, weight and position written
    if op == "append":
        n = case["tokens"] * case["heads"] * d
        return {"bytes": move + 2 * n * es, "flops": 3 * case["rotary"] * (rows + case["tokens"] * case["heads"])}
    if case["one"]:
        held = case["batch"] * case["kv_heads"]
        return {"bytes": move + held * (8 * (case["budget"] + 1) + 4 * d * es + 16), "flops": 2 * held * case["budget"]}
    # a prompt of n rows keeps the budget: of the rows below it, the share that goes is filled from above
    each = case["tokens"] / case["batch"]
    holes = case["budget"] * (1 - case["budget"] / each) * case["batch"] if each > case["budget"] else 0
    return {"bytes": move + 8 * rows + int(holes * case["kv_heads"] * (4 * d * es + 16)), "flops": 2 * rows}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _cut(tokens, batch, gen):
    """Prefix sums of a ragged split of `tokens` into `batch` prompts of one token at least: always the same lengths, in
    another order."""
    share = torch.linspace(0.1, 1.1, batch, dtype=torch.float64)
    n = (share / share.sum() * (tokens - batch)).floor().to(torch.int64) + 1
    n[-1] += tokens - int(n.sum())
    return [0] + n[torch.randperm(batch, generator=gen)].cumsum(0).tolist()


def _cache(case, batch, longest, g, gen, dt):
    """Empty-looking pages in no order, with a few more than are used."""
    page, heads, d = case["page"], case["kv_heads"], case["dim"]
    each = -(-longest // page)
    pages = batch * each + 3
    table = torch.randperm(pages, generator=gen)[: batch * each].reshape(batch, each).to(torch.int32).to(DEV)
    shape = (pages, heads, page)
    return {"k_pages": torch.randn(*shape, d, device=DEV, generator=g, dtype=dt),
            "v_pages": torch.randn(*shape, d, device=DEV, generator=g, dtype=dt),
            "weight": torch.randn(shape, device=DEV, generator=g).mul_(2).exp_(),
            "pos": torch.zeros(shape, device=DEV, dtype=torch.int32),
            "page_table": table, "counts": torch.zeros(2, batch, device=DEV, dtype=torch.int32)}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    dt, d = DTYPES[case["dtype"]], case["dim"]
    s = {"case": case}

    def rnd(*shape):
        return torch.randn(*shape, device=DEV, generator=g, dtype=dt)

    if case["op"] == "rope":
        t, h = case["tokens"], case["heads"]
        s["x"] = rnd(t, h + case["extra"], d)[:, :h]
        start = torch.randint(0, max(1, case["max_pos"] - t + 1), (1,), generator=gen).item()
        s["positions"] = torch.arange(start, start + t, device=DEV, dtype=torch.int32)
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["dy"] = rnd(t, h, d)
    elif case["op"] == "append":
        b, t = case["batch"], case["tokens"]
        cu = list(range(b + 1)) if case["one"] else _cut(t, b, gen)
        longest = case["seen"] + max(y - x for x, y in zip(cu, cu[1:]))
        s.update(_cache(case, b, longest, g, gen, dt))
        s["cu"] = None if case["one"] else torch.tensor(cu, dtype=torch.int32, device=DEV)
        s["before"] = torch.full((2, b), case["seen"], dtype=torch.int32, device=DEV)
        if case["one"]:
            s["before"] -= torch.randint(0, case["seen"] // 2 + 1, (b,), generator=gen).to(torch.int32).to(DEV)
        s["q"], s["k"], s["v"] = rnd(t, case["heads"], d), rnd(t, case["kv_heads"], d), rnd(t, case["kv_heads"], d)
    elif case["op"] == "attend":
        b, lens = case["batch"], _lengths(case)
        s.update(_cache(case, b, max(lens), g, gen, dt))
        order = torch.randperm(b, generator=gen)
        s["counts"].copy_(torch.tensor(lens, dtype=torch.int32)[order].expand(2, b))
        s["q"] = rnd(b, case["heads"], d) * 2
        s["valid"] = None
        if case["masked"]:  # padding inside the prompt; the newest row always counts
            s["valid"] = torch.rand(b, max(lens), device=DEV, generator=g) > 0.1
            s["valid"].scatter_(1, s["counts"][0].long()[:, None] - 1, True)
    else:
        b, t = case["batch"], case["tokens"]
        cu = list(range(b + 1)) if case["one"] else _cut(t, b, gen)
        longest = case["budget"] + 1 if case["one"] else max(y - x for x, y in zip(cu, cu[1:]))
        s.update(_cache(case, b, longest, g, gen, dt))
        s["cu"] = None if case["one"] else torch.tensor(cu, dtype=torch.int32, device=DEV)
        s["k"], s["v"] = rnd(t, case["kv_heads"], d), rnd(t, case["kv_heads"], d)
        s["new_weight"] = None
        if case["one"]:  # at the budget, rows of each head in an order of their own out of four times as many tokens
            seen = 4 * case["budget"]
            held = torch.rand(b, case["kv_heads"], seen, device=DEV, generator=g).argsort(-1)[..., : case["budget"]]
            at = torch.arange(case["budget"], device=DEV)
            pg = s["page_table"][:, at // case["page"]].long()
            s["pos"][pg, :, (at % case["page"])[None]] = held.transpose(1, 2).to(torch.int32)
            s["counts"][0], s["counts"][1] = case["budget"], seen
        else:  # what the prefill's attention gave each key
            s["new_weight"] = torch.randn(t, case["kv_heads"], device=DEV, generator=g).mul_(2).exp_()
    if own:
        pkg = _package()
        if "rotary" in case:
            s["freqs"] = pkg.RopeFrequencies(case["rotary"], case["base"], layout=case["layout"],
                                             scaling=None if case["scaling"] == "none" else case["scaling"],
                                             factor=case["factor"], original_len=case["original"] or None, device=DEV)
        if case["op"] != "rope":
            s["cache"] = pkg.PagedKVCache(s["k_pages"], s["v_pages"], s["page_table"], s["counts"], pos=s["pos"],
                                          weight=s["weight"])
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------


def _frequencies(case):
    """(angle per position of each pair, fp64; factor on cos and sin)."""
    r, base, f = case["rotary"], case["base"], case["factor"]
    if case["scaling"] == "ntk":
        base = base * f ** (r / (r - 2))
    i = torch.arange(r // 2, dtype=torch.float64, device=DEV)
    inv = base ** (-2 * i / r)
    if case["scaling"] == "linear":
        return inv / f, 1.0
    if case["scaling"] == "yarn":
        low = max(math.floor(r * math.log(case["original"] / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
        high = min(math.ceil(r * math.log(case["original"] / (2 * math.pi)) / (2 * math.log(base))), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _rotate(case, x, positions, transpose=False):
    """Rotates the first `rotary` values of each head: x [tokens, heads, dim], positions [tokens]."""
    r = case["rotary"]
    inv, mag = _frequencies(case)
    angle = positions.double()[:, None] * inv
    c, s = (angle.cos() * mag).float()[:, None], (angle.sin() * mag).float()[:, None]
    s = -s if transpose else s
    y = x.float().clone()
    if case["layout"] == "half":
        a, b = x[..., : r // 2].float(), x[..., r // 2 : r].float()
        y[..., : r // 2], y[..., r // 2 : r] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:r:2].float(), x[..., 1:r:2].float()
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    return y.to(x.dtype)


def _plain_append(s, weight=None):
    """Rows of the new tokens behind each sequence's last; the rotated q."""
    case, table, counts = s["case"], s["page_table"], s["counts"]
    t, page = s["k"].shape[0], case["page"]
    at = torch.arange(t, device=DEV)
    if s["cu"] is None:
        seq, off = at, torch.zeros_like(at)
        n = torch.ones_like(counts[0])
    else:
        seq = torch.searchsorted(s["cu"][1:].contiguous(), at.to(torch.int32), right=True)
        off, n = at - s["cu"][seq], s["cu"][1:] - s["cu"][:-1]
    row, where = counts[0][seq] + off, counts[1][seq] + off
    pg, line = table[seq, row // page].long(), (row % page).long()
    q = None
    k = s["k"]
    if "rotary" in case:
        k, q = _rotate(case, k, where), _rotate(case, s["q"], where)
    s["k_pages"][pg, :, line] = k
    s["v_pages"][pg, :, line] = s["v"]
    s["pos"][pg, :, line] = where.to(torch.int32)[:, None].expand(-1, case["kv_heads"])
    s["weight"][pg, :, line] = torch.zeros(t, case["kv_heads"], device=DEV) if weight is None else weight
    counts += n
    return q


def _plain_attend(s):
    case, q, lens = s["case"], s["q"], s["counts"][0]
    b, hq, d = q.shape
    hk, page = case["kv_heads"], case["page"]
    at = torch.arange(case["longest"], device=DEV)
    pg, line = s["page_table"][:, at // page].long(), (at % page)[None].expand(b, -1)
    k, v = s["k_pages"][pg, :, line].float(), s["v_pages"][pg, :, line].float()  # [b, rows, hk, d]
    x = torch.matmul(q.float().reshape(b, hk, hq // hk, d), k.permute(0, 2, 3, 1)) / math.sqrt(d)
    live = at[None] < lens[:, None]
    if s["valid"] is not None:
        live = live & s["valid"]
    x = torch.where(live[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    p = e / total
    v = torch.where(live[:, :, None, None], v, 0.0)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).reshape(b, hq, d).to(q.dtype)
    if case["track"]:
        add = torch.where(live[:, None], p.sum(2), 0.0).transpose(1, 2)  # [b, rows, hk]
        keep = live.reshape(-1)
        pg, line = pg.reshape(-1)[keep], line.reshape(-1)[keep]
        s["weight"][pg, :, line] += add.reshape(-1, hk)[keep]
    return out, (total.log() + top).reshape(b, hq)


def _plain_evict(s):
    """Each head gives up its lowest-weighted rows beyond the budget; rows from above fill the holes in order."""
    case, counts, page = s["case"], s["counts"], s["case"]["page"]
    hk, budget = case["kv_heads"], case["budget"]
    at = torch.arange(s["page_table"].shape[1] * page, device=DEV)
    pg, line = s["page_table"][:, at // page].long(), (at % page)[None]
    w, pos = s["weight"][pg, :, line].transpose(1, 2), s["pos"][pg, :, line].transpose(1, 2)  # [b, hk, rows]
    lens, seen = counts[0].long()[:, None, None], counts[1].long()[:, None, None]
    left = lens.clamp(max=budget)
    w = torch.where((pos >= seen - case["recent"]) | (pos < case["sinks"]), math.inf, w)
    live = at < lens
    order = torch.where(live, w, math.inf).sort(dim=-1, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order))
    gone = live & (rank < lens - left)
    hole, tail = gone & (at < left), live & ~gone & (at >= left)
    far = at.shape[0]
    src = torch.where(tail, at, far).sort(-1).values
    dst = torch.where(hole, at, far).sort(-1).values
    used = dst < far
    b_at, h_at = (torch.arange(n, device=DEV) for n in (counts.shape[1], hk))
    b_at, h_at = (x.expand_as(dst)[used] for x in (b_at[:, None, None], h_at[None, :, None]))
    src, dst = src[used], dst[used]
    ps, pd = s["page_table"][b_at, src // page].long(), s["page_table"][b_at, dst // page].long()
    for name in ("k_pages", "v_pages", "weight", "pos"):
        s[name][pd, h_at, dst % page] = s[name][ps, h_at, src % page]
    counts[0].clamp_(max=budget)


def _state(s):
    return {n: s[n] for n in ("k_pages", "v_pages", "weight", "pos", "counts")}


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "rope":
        if not case["grad"]:
            return _package().rope(s["x"], s["positions"], s["freqs"]) if own else _rotate(case, s["x"], s["positions"])
        if own:
            y = _package().rope(s["x"], s["positions"], s["freqs"])
            return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]
        return (_rotate(case, s["x"].detach(), s["positions"]),
                _rotate(case, s["dy"], s["positions"], transpose=True))
    if op == "append":
        s["counts"].copy_(s["before"])  # other sequences take the pages
        if own:
            q = s["cache"].append(s["k"], s["v"], q=s["q"], freqs=s["freqs"], cu_tokens=s["cu"])
        else:
            q = _plain_append(s)
        return {"q": q, **_state(s)}
    if op == "attend":
        if own:
            out, lse = s["cache"].attend(s["q"], key_valid=s["valid"], track=case["track"], return_lse=True)
        else:
            out, lse = _plain_attend(s)
        return {"out": out, "lse": lse, **({"weight": s["weight"]} if case["track"] else {})}
    if not case["one"]:
        s["counts"].zero_()  # new prompts take the pages
    if own:
        s["cache"].append(s["k"], s["v"], cu_tokens=s["cu"], weight=s["new_weight"])
        s["cache"].evict(case["budget"], recent=case["recent"], sinks=case["sinks"])
    else:
        _plain_append(s, s["new_weight"])
        _plain_evict(s)
    return _state(s)


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------


def _turned(case, x, positions, sign=1.0):
    """x [n, heads, dim] at positions [n] as complex numbers times magnitude * exp(i * sign * angle)."""
    r, f = case["rotary"], case["factor"]
    k = torch.arange(0, r, 2, dtype=torch.float64, device=x.device)
    base = case["base"] * (f ** (r / (r - 2)) if case["scaling"] == "ntk" else 1.0)
    w = torch.exp(-math.log(base) * k / r)
    m = 1.0
    if case["scaling"] == "linear":
        w = w / f
    elif case["scaling"] == "yarn":
        turns = [math.log(case["original"] / (n * 2 * math.pi)) * r / (2 * math.log(base)) for n in (32, 1)]
        lo, hi = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), r - 1)
        mix = torch.clamp((k / 2 - lo) / max(hi - lo, 0.001), 0, 1)
        w, m = w * (mix / f + 1 - mix), 1.0 + 0.1 * math.log(f)
    a = sign * positions.double()[:, None, None] * w
    z = torch.polar(torch.full_like(a, m), a)
    y = x.detach().double().clone()
    if case["layout"] == "half":
        c = torch.complex(y[..., : r // 2], y[..., r // 2 : r]) * z
        y[..., :r] = torch.cat([c.real, c.imag], -1)
    else:
        c = torch.view_as_complex(y[..., :r].reshape(*y.shape[:-1], r // 2, 2).contiguous()) * z
        y[..., :r] = torch.view_as_real(c).flatten(-2)
    return y


def _exact_append(s, weight=None):
    """The cache after the append, as 64-bit copies, and the rotated q; one sequence at a time."""
    case = s["case"]
    page, t = case["page"], s["k"].shape[0]
    cu = list(range(t + 1)) if s["cu"] is None else s["cu"].tolist()
    lens, seen = s["counts"].tolist()
    c = {"k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double(), "weight": s["weight"].double(),
         "pos": s["pos"].clone()}
    q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV) if "rotary" in case else None
    for b in range(len(lens)):
        lo, hi = cu[b], cu[b + 1]
        rows = torch.arange(lens[b], lens[b] + hi - lo, device=DEV)
        where = torch.arange(seen[b], seen[b] + hi - lo, device=DEV)
        pg, line = s["page_table"][b].long()[rows // page], rows % page
        k = s["k"][lo:hi].double()
        if q is not None:
            k, q[lo:hi] = _turned(case, s["k"][lo:hi], where), _turned(case, s["q"][lo:hi], where)
        for h in range(case["kv_heads"]):
            c["k_pages"][pg, h, line] = k[:, h]
            c["v_pages"][pg, h, line] = s["v"][lo:hi, h].double()
            c["pos"][pg, h, line] = where.to(torch.int32)
            c["weight"][pg, h, line] = 0.0 if weight is None else weight[lo:hi, h].double()
        lens[b], seen[b] = lens[b] + hi - lo, seen[b] + hi - lo
    c["counts"] = torch.tensor([lens, seen], dtype=torch.int32, device=DEV)
    return c, q


def _exact_evict(s, c):
    case = s["case"]
    page, lens, seen = case["page"], *c["counts"].tolist()
    for b, n in enumerate(lens):
        left = min(n, case["budget"])
        if n == left:
            continue
        rows = torch.arange(n, device=DEV)
        pg, line = s["page_table"][b].long()[rows // page], rows % page
        for h in range(case["kv_heads"]):
            p, w = c["pos"][pg, h, line], c["weight"][pg, h, line].clone()
            w[(p >= seen[b] - case["recent"]) | (p < case["sinks"])] = math.inf
            stays = torch.ones(n, dtype=torch.bool, device=DEV)
            stays[w.sort(dim=0, stable=True).indices[: n - left]] = False
            dst, src = (~stays[:left]).nonzero()[:, 0], stays[left:].nonzero()[:, 0] + left
            for x in (c["k_pages"], c["v_pages"], c["weight"], c["pos"]):
                x[pg[dst], h, line[dst]] = x[pg[src], h, line[src]]
        lens[b] = left
    c["counts"] = torch.tensor([lens, seen], dtype=torch.int32, device=DEV)


def _exact_attend(s):
    case, page = s["case"], s["case"]["page"]
    b, hq, d = s["q"].shape
    hk = case["kv_heads"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=DEV)
    lse = torch.zeros(b, hq, dtype=torch.float64, device=DEV)
    weight = s["weight"].double()
    for i, n in enumerate(s["counts"][0].tolist()):
        rows = torch.arange(n, device=DEV)
        if s["valid"] is not None:
            rows = rows[s["valid"][i, :n]]
        pg, line = s["page_table"][i].long()[rows // page], rows % page
        for h in range(hk):
            heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
            x = s["q"][i, heads].double() @ s["k_pages"][pg, h, line].double().T * d**-0.5
            lse[i, heads] = torch.logsumexp(x, -1)
            p = (x - lse[i, heads, None]).exp()
            out[i, heads] = p @ s["v_pages"][pg, h, line].double()
            weight[pg, h, line] += p.sum(0)
    return {"out": out, "lse": lse, **({"weight": weight} if case["track"] else {})}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        y = _turned(case, s["x"], s["positions"])
        return (y, _turned(case, s["dy"], s["positions"], -1.0)) if case["grad"] else y
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        s["counts"].copy_(s["before"])
        c, q = _exact_append(s)
        return {"q": q, **c}
    if not case["one"]:
        s["counts"].zero_()
    c, _ = _exact_append(s, s["new_weight"])
    _exact_evict(s, c)
    return c
