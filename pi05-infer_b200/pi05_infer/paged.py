"""Text decoding on a paged key-value cache: rotary positions, append, single-token
attention, and eviction by accumulated attention weight.

The engine's own loop (``expert.py``) keeps one dense cache per observation; a program
that decodes text next to it -- tokens one at a time, many sequences of different
lengths, long contexts -- keeps its keys and values in pages::

    freqs = RopeFrequencies(256, device="cuda")
    cache = PagedKVCache.allocate(num_pages=512, page_size=64, n_kv_heads=1, head_dim=256, batch=4,
                                  pages_per_seq=32, device="cuda")
    cache.page_table.copy_(...)                     # which pages each sequence owns
    cache.append(k, v, cu_tokens=cu, freqs=freqs)   # prompts, ragged
    q = cache.append(k1, v1, q=q1, freqs=freqs)     # then one token of each sequence
    out = cache.attend(q, track=True)
    cache.evict(budget=1024, recent=128, sinks=4)

Rotary embedding: the reference's ``modeling_gemma.py:151-216`` (half layout, no
scaling); the cache has no counterpart there.  Calls run on the current stream of the
tensors' device and never synchronise; calls on one cache are to be ordered on one
stream (or by events).  Everything can be captured in a CUDA graph; ``torch.jit.trace`` and
``make_fx``, which see none of these calls, are refused.
"""

from __future__ import annotations

import ctypes
import math
import struct
from decimal import Decimal, localcontext
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib

_P = ctypes.c_void_p
_I = ctypes.c_int
_L = ctypes.c_longlong
_Z = ctypes.c_size_t
_F = ctypes.c_float

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITIONS = (torch.int32, torch.int64)


class Pi05Rotary(ctypes.Structure):
    _fields_ = [("turns", _P), ("rotary_dim", _I), ("interleaved", _I), ("magnitude", _F)]


class Pi05RopeArgs(ctypes.Structure):
    _fields_ = [
        ("x", _P), ("out", _P), ("positions", _P), ("x_token_stride", _L), ("x_head_stride", _L),
        ("out_token_stride", _L), ("out_head_stride", _L), ("dtype", _I), ("tokens", _I), ("heads", _I),
        ("head_dim", _I), ("positions_i64", _I), ("transpose", _I),
    ]


class Pi05PagedCache(ctypes.Structure):
    _fields_ = [
        ("k_pages", _P), ("v_pages", _P), ("page_stride", _L), ("head_stride", _L), ("row_stride", _L),
        ("weight", _P), ("pos", _P), ("page_table", _P), ("counts", _P),
        ("dtype", _I), ("num_pages", _I), ("page_size", _I), ("n_kv_heads", _I), ("head_dim", _I),
        ("batch", _I), ("pages_per_seq", _I), ("table_pitch", _I),
        ("workspace", _P), ("workspace_bytes", _Z),
    ]


class Pi05PagedAppend(ctypes.Structure):
    _fields_ = [
        ("k", _P), ("v", _P), ("k_token_stride", _L), ("k_head_stride", _L), ("v_token_stride", _L),
        ("v_head_stride", _L), ("q", _P), ("q_out", _P), ("q_token_stride", _L), ("q_head_stride", _L),
        ("tokens", _I), ("n_q_heads", _I), ("cu_tokens", _P), ("new_weight", _P), ("rotary", _P),
    ]


class Pi05PagedAttention(ctypes.Structure):
    _fields_ = [
        ("q", _P), ("out", _P), ("lse", _P), ("key_valid", _P), ("q_token_stride", _L), ("q_head_stride", _L),
        ("valid_pitch", _L), ("valid_rows", _I), ("n_q_heads", _I), ("scale", _F), ("track", _I), ("scratch", _P), ("scratch_bytes", _Z),
    ]


# The argument structs as bytes: packing one takes a fifth of the time that filling a ctypes
# structure does, and these calls come once for every token.
_ROPE_ARGS = struct.Struct("@3P4q6i")
_APPEND_ARGS = struct.Struct("@2P4q2P2q2i3P")
_ATTEND_ARGS = struct.Struct("@4P3q2ifiPN")

_lib.SIGNATURES.update({
    "pi05_rope": (_I, [_P, _P, _P]),
    "pi05_paged_workspace_bytes": (_Z, [_P]),
    "pi05_paged_append": (_I, [_P, _P, _P]),
    "pi05_paged_attention_scratch_bytes": (_Z, [_P, _I, _I]),
    "pi05_paged_attention": (_I, [_P, _P, _P]),
    "pi05_paged_evict": (_I, [_P, _I, _I, _I, _P]),
})
_fns = {}


def _fn(name: str):
    f = _fns.get(name)
    if f is None:
        f = getattr(_lib.lib(), name)
        f.restype, f.argtypes = _lib.SIGNATURES[name]
        _fns[name] = f
    return f


# The current stream's handle and the current device without the objects around them.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_raw_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


# Whether torch records operators: what there is to ask in 0.2 us, where get_proxy_mode() and
# torch.jit.is_tracing() take 0.5.
_is_tracing = getattr(torch._C, "_is_tracing", None) or torch.jit.is_tracing
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None) or (lambda: 1)
_early_modes = (torch._ops.mode_stack_state_for_pre_dispatch().count
                if hasattr(torch._ops, "mode_stack_state_for_pre_dispatch") else (lambda: 1))


def _run(name: str, index: int, *args) -> None:
    """Calls the library on the current stream of device ``index``, whichever device is current.

    Refused where torch records the operators that run (``torch.jit.trace``, ``make_fx``): a call of the
    library leaves nothing in such a record, whose replay would return memory that nobody wrote.
    """
    if _is_tracing() or (_modes() or _early_modes()) and get_proxy_mode() is not None:
        raise ValueError(f"{name} cannot be recorded by torch.jit.trace or make_fx (a CUDA graph can hold it)")
    if index == _raw_device():
        rc = _fn(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = _fn(name)(*args, _raw_stream(index))
    if rc != _lib.PI05_OK:
        raise _lib.Pi05Error(name, rc, _lib.last_error())


_increment_version = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version


def _wrote(tensors) -> None:
    """Tells torch, which cannot see it, that the library wrote into ``tensors``: a graph that saved one of them is
    then refused its backward pass instead of reading the new values."""
    _increment_version(tensors)


def _wants_grad(t: torch.Tensor) -> bool:
    """Whether a derivative of what is made of ``t`` is wanted, in reverse or in forward mode (a tangent, which
    ``requires_grad`` does not tell)."""
    return (t.requires_grad and torch.is_grad_enabled()) or \
        (forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None)


def _strides(t: torch.Tensor):
    """``t``'s strides, with those of dimensions of one element, which mean nothing, as if it were dense there."""
    strides, dense = list(t.stride()), 1
    for i in reversed(range(t.dim())):
        if t.shape[i] == 1:
            strides[i] = dense
        dense = max(dense, strides[i] * t.shape[i])
    return strides


def _cuda(device) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"expected a CUDA device, got {device} (pi05_infer has no CPU fallback)")
    return device if device.index is not None else torch.device("cuda", torch.cuda.current_device())


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


_ONE = 1 << 128
_PER_RAD = 0x28be60db9391054a7f09d5f47d4d3770  # 2^128 / (2 pi): turns of a radian


def _exact_frequencies(rotary_dim, base, scaling, factor, original_len, beta_fast, beta_slow):
    """Rad per position of each pair, in units of 2^-128 (a 64-bit float's 53 bits would show from position 10^8 on), and
    the factor on cos and sin."""
    base, factor = float(base), float(factor)
    num, den = factor.as_integer_ratio()
    with localcontext() as context:
        context.prec = 40
        ratio = Decimal(base) ** (Decimal(-2) / rotary_dim)
        if scaling == "ntk":  # (base factor^(rotary_dim / (rotary_dim - 2)))^(-2 / rotary_dim)
            ratio *= Decimal(factor) ** (Decimal(-2) / (rotary_dim - 2))
        ratio = int(ratio * _ONE)
    inv_freq = [_ONE]
    while len(inv_freq) < rotary_dim // 2:
        inv_freq.append(inv_freq[-1] * ratio >> 128)
    if scaling == "linear":
        return [f * den // num for f in inv_freq], 1.0
    if scaling != "yarn":
        return inv_freq, 1.0

    def pair(turns):  # number (not whole) of the pair that turns so often within original_len
        return rotary_dim * math.log(original_len / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rotary_dim - 1)
    scale, width = (1, high - low) if high > low else (1000, 1)  # at least a thousandth of a pair wide
    ramp = [min(max((i - low) * scale, 0), width) for i in range(rotary_dim // 2)]
    return [f * (r * den + (width - r) * num) // (width * num) for f, r in zip(inv_freq, ramp)], 0.1 * math.log(factor) + 1.0


def _floats(inv_freq):
    return [f / _ONE for f in inv_freq]


def _pair_frequencies(*args):
    """As 64-bit floats."""
    inv_freq, magnitude = _exact_frequencies(*args)
    return _floats(inv_freq), magnitude


def _turns(inv_freq):
    """Fractions of a turn per position in units of 2^-64, rounded (below one half: every frequency is at most 1 rad)."""
    return [((f if isinstance(f, int) else int(f * _ONE)) * _PER_RAD + (1 << 191)) >> 192 for f in inv_freq]


class RopeFrequencies:
    """What each pair of a head turns by per position, as the kernels take it.

    Pair ``i`` of the first ``rotary_dim`` values of a head turns by ``base ** (-2 i /
    rotary_dim)`` rad per position.  ``layout``: ``"half"`` pairs value ``i`` with ``i +
    rotary_dim / 2`` (``modeling_gemma.py:184-216``), ``"interleaved"`` ``2 i`` with ``2 i +
    1``.  ``scaling`` for contexts longer than the trained ``original_len``, by ``factor``:

    * ``"linear"``: every frequency divided by ``factor`` (position interpolation);
    * ``"ntk"``: ``base * factor ** (rotary_dim / (rotary_dim - 2))``;
    * ``"yarn"``: pairs that turn less than ``beta_slow`` times within ``original_len`` are
      divided by ``factor``, those over ``beta_fast`` times are kept, a linear ramp over the pair
      number between; cos and sin times ``0.1 ln(factor) + 1``.

    The device table holds fractions of a turn in 64-bit fixed point, each rounded once: an angle is
    off by 2^-65 turn for each position, which is nothing to its fp32 cos and sin up to position 2^36.
    """

    def __init__(self, rotary_dim: int, base: float = 10000.0, *, layout: str = "half", scaling: Optional[str] = None,
                 factor: float = 1.0, original_len: Optional[int] = None, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, device="cuda"):
        if rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > 512:
            raise ValueError(f"rotary_dim {rotary_dim} is not an even number of 2..512")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout {layout!r} is not 'half' or 'interleaved'")
        if scaling not in (None, "linear", "ntk", "yarn"):
            raise ValueError(f"scaling {scaling!r} is not None, 'linear', 'ntk' or 'yarn'")
        if not base > 1 or not math.isfinite(base):
            raise ValueError(f"base {base} is not above 1")
        if scaling is not None and not (factor >= 1 and math.isfinite(factor)):
            raise ValueError(f"factor {factor} is not 1 or more")
        if scaling == "ntk" and rotary_dim == 2:
            raise ValueError("'ntk' scaling needs rotary_dim > 2")
        if scaling == "yarn" and (original_len is None or original_len <= 0 or not beta_fast > beta_slow > 0):
            raise ValueError("'yarn' scaling needs original_len and beta_fast > beta_slow > 0")
        self.rotary_dim, self.layout = rotary_dim, layout
        exact, self.magnitude = _exact_frequencies(rotary_dim, base, scaling, factor, original_len, beta_fast, beta_slow)
        self.inv_freq = _floats(exact)
        turns = _turns(exact)
        self.device = _cuda(device)
        self.turns = torch.tensor(turns, dtype=torch.int64).to(self.device)
        self._index = self.device.index
        self._c = Pi05Rotary(self.turns.data_ptr(), rotary_dim, int(layout == "interleaved"), self.magnitude)
        self._at = ctypes.addressof(self._c)


def _rope(x, positions, freqs, out, transpose):
    """``out`` None: with ``x``'s strides, or dense where torch cannot keep them (views that overlap) and would part a
    head's values."""
    tokens, heads, dim = x.shape
    xt, xh, _ = x.stride()
    if out is None:
        out = torch.empty_like(x)
        ot, oh, part = out.stride()
        if part != 1:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
            ot, oh, _ = out.stride()
    else:
        ot, oh, _ = out.stride()
    if heads == 0:
        return out
    _run("pi05_rope", freqs._index, _ROPE_ARGS.pack(
        x.data_ptr(), out.data_ptr(), positions.data_ptr(), xt, xh, ot, oh, _DTYPES[x.dtype], tokens, heads, dim,
        positions.dtype == torch.int64, transpose), freqs._at)
    return out


def _rows_apart(x: torch.Tensor) -> bool:
    """Whether the heads of ``x``, contiguous ones, lie apart: tokens before heads in memory, or after."""
    (tokens, heads, dim), (t, h, _) = x.shape, x.stride()
    return (heads <= 1 or h >= dim) and (tokens <= 1 or t >= max(heads - 1, 0) * h + dim) or \
        (tokens <= 1 or t >= dim) and (heads <= 1 or h >= max(tokens - 1, 0) * t + dim)


def _leaf_node(x: torch.Tensor):
    """The node that accumulates leaf ``x``'s gradient, marked with the stream it was first seen on.

    Torch makes it with the first graph that uses the leaf and keeps it as long as any lives; a backward
    pass waits for its stream, which a capture on another stream cannot (torch then breaks the capture off
    and leaves its random generator in it).  So a captured call is refused while such a graph is alive;
    torch does not say on which stream other operators made one.
    """
    node = torch.autograd.graph.get_gradient_edge(x).node
    stream = _raw_stream(x.get_device())
    if node.metadata.setdefault("pi05_stream", stream) != stream and torch.cuda.is_current_stream_capturing():
        raise ValueError("x is a leaf that an earlier graph, made on another stream, still uses: drop that graph "
                         "before capturing this call")
    return node


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, freqs, transpose):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.freqs, ctx.transpose = freqs, transpose
        return _rope(x, positions, freqs, None, transpose)

    @staticmethod
    def backward(ctx, g):
        (positions,) = ctx.saved_tensors
        g = g if g.stride(-1) == 1 else g.contiguous()
        if torch.is_grad_enabled():  # a gradient of the gradient is wanted
            gx = _Rope.apply(g, positions, ctx.freqs, not ctx.transpose)
        else:
            gx = _rope(g, positions, ctx.freqs, None, not ctx.transpose)
        return gx, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        (positions,) = ctx.saved_tensors
        tangent = tangent if tangent.stride(-1) == 1 else tangent.contiguous()
        return _Rope.apply(tangent, positions, ctx.freqs, ctx.transpose)


def rope(x: torch.Tensor, positions: torch.Tensor, freqs: RopeFrequencies, *, transpose: bool = False,
         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` ``[tokens, heads, dim]`` with the first ``freqs.rotary_dim`` values of each head rotated
    to ``positions`` ``[tokens]`` (int32 or int64, any sign).

    bf16, fp16 or fp32, fp32 math, one rounding.  Any token and head strides (a q|k|v row's q and k
    heads in one call, say, or views that overlap); values of a head contiguous.  ``out`` may be ``x``
    (in place), but not overlap it otherwise, nor itself.  ``transpose`` turns backwards.
    Differentiable in ``x``, in reverse and forward mode, when ``out`` is not given.  A captured call
    with a leaf ``x`` is refused while a graph that this function made of it on another stream is
    alive; drop graphs that other operators made of it before such a capture.
    """
    if x.dim() != 3 or x.dtype not in _DTYPES or not x.is_cuda or x.stride(2) != 1:
        raise ValueError("x must be a [tokens, heads, dim] CUDA tensor, bf16, fp16 or fp32, contiguous in dim")
    index, (tokens, _, dim) = x.get_device(), x.shape
    if positions.dim() != 1 or positions.shape[0] != tokens or positions.dtype not in _POSITIONS or \
            positions.get_device() != index or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32 or int64 [tokens] on x's device")
    if freqs._index != index:
        raise ValueError(f"the frequencies are on {freqs.device}, x is on {x.device}")
    if freqs.rotary_dim > dim:
        raise ValueError(f"rotary_dim {freqs.rotary_dim} is more than the head's {dim} values")
    grad = _wants_grad(x)
    if out is None:
        if grad:
            # alive until the new graph holds it
            node = _leaf_node(x) if x.is_leaf and x.requires_grad and torch.is_grad_enabled() else None
            y = _Rope.apply(x, positions, freqs, bool(transpose))
            del node
            return y
    elif grad:
        raise ValueError("out= is not differentiable")
    elif out.shape != x.shape or out.dtype != x.dtype or out.get_device() != index or out.stride(2) != 1 or \
            _wants_grad(out):
        raise ValueError("out must have x's shape, type and device, contiguous in dim, and need no gradient")
    elif not _rows_apart(out):
        raise ValueError("out's heads overlap")
    y = _rope(x, positions, freqs, out, bool(transpose))
    if out is not None:
        _wrote((out,))
    return y


# ---------------------------------------------------------------------------
# the paged cache
# ---------------------------------------------------------------------------


class PagedKVCache:
    """Keys and values of ``batch`` sequences in pages.

    ``k_pages`` / ``v_pages`` ``[num_pages, n_kv_heads, page_size, head_dim]`` (bf16 or fp16, same
    strides, rows on 16-byte boundaries), ``page_table`` ``[batch, pages_per_seq]`` int32, ``counts``
    ``[2, batch]`` int32 (rows held; tokens seen, which is the next token's position), and for
    eviction ``weight`` (fp32) and ``pos`` (int32) ``[num_pages, n_kv_heads, page_size]``.  Row ``r``
    of sequence ``b`` is line ``r % page_size`` of page ``page_table[b, r // page_size]``.  The
    tensors stay the caller's: who owns which page, and resetting or truncating a sequence (``counts``),
    is done by writing to them, not by putting others in their place, which is refused.

    The table is read on the device.  A page number outside the cache, or a row beyond the table,
    is skipped or masked and sets ``PI05_DEV_BAD_INDEX`` (0x20) in :meth:`read_status`.  A page that a
    call writes (:meth:`append`, :meth:`evict`, :meth:`attend` with ``track``) stands once in the
    table, with one sequence; pages that are only read may be shared.
    """

    _FIXED = frozenset(("k_pages", "v_pages", "page_table", "counts", "weight", "pos", "workspace"))

    def __setattr__(self, name, value):
        if name in self._FIXED and name in self.__dict__:  # the library has the first one's address
            raise AttributeError(f"{name} stays the tensor that the cache was built with: write into it, or build "
                                 "another cache")
        super().__setattr__(name, value)

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, counts: torch.Tensor, *,
                 weight: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None):
        if k_pages.dim() != 4 or k_pages.dtype not in (torch.bfloat16, torch.float16) or not k_pages.is_cuda:
            raise ValueError("k_pages must be a [pages, kv_heads, page_size, dim] CUDA tensor, bf16 or fp16")
        device = k_pages.device
        strides = _strides(k_pages)
        if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != device or \
                _strides(v_pages) != strides or strides[3] != 1:
            raise ValueError("v_pages must match k_pages (shape, type, device, strides; rows contiguous)")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != device or \
                _strides(page_table)[1] != 1:
            raise ValueError("page_table must be int32 [batch, pages_per_seq] on the cache's device, rows contiguous")
        if counts.shape != (2, page_table.shape[0]) or counts.dtype != torch.int32 or counts.device != device or \
                not counts.is_contiguous():
            raise ValueError("counts must be contiguous int32 [2, batch] on the cache's device")
        for t, dt, name in ((weight, torch.float32, "weight"), (pos, torch.int32, "pos")):
            if t is not None and (t.shape != k_pages.shape[:3] or t.dtype != dt or t.device != device or
                                  not t.is_contiguous()):
                raise ValueError(f"{name} must be contiguous {dt} {list(k_pages.shape[:3])} on the cache's device")
        self.k_pages, self.v_pages, self.page_table, self.counts = k_pages, v_pages, page_table, counts
        self.weight, self.pos, self.device, self.dtype = weight, pos, device, k_pages.dtype
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k_pages.shape
        self.batch, self.pages_per_seq = page_table.shape

        def p(t):
            return None if t is None else t.data_ptr()

        self._c = Pi05PagedCache(
            p(k_pages), p(v_pages), *strides[:3], p(weight), p(pos), p(page_table), p(counts),
            _DTYPES[self.dtype], self.num_pages, self.page_size, self.n_kv_heads, self.head_dim, self.batch,
            self.pages_per_seq, _strides(page_table)[0], None, 0)
        self._at, self._index = ctypes.addressof(self._c), device.index
        self._state = tuple(t for t in (k_pages, v_pages, counts, weight, pos) if t is not None)
        nbytes = _fn("pi05_paged_workspace_bytes")(self._at)
        # What else the library asks of a cache (head sizes, alignment, 32-bit ranges), before memory is taken: an
        # append of no tokens checks it and runs nothing; the workspace is not looked at.
        self._c.workspace, self._c.workspace_bytes = 256, nbytes
        if _fn("pi05_paged_append")(self._at, _APPEND_ARGS.pack(*[0] * 12, counts.data_ptr(), 0, 0), None) != _lib.PI05_OK:
            raise ValueError(f"not a cache that the library takes: {_lib.last_error()}")
        # status word, ticket and the eviction's lists; zeroed once
        self.workspace = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        self._c.workspace, self._c.workspace_bytes = self.workspace.data_ptr(), nbytes
        # (heads, track): bytes of scratch, and one-element tensors with the shapes of scratch and lse
        self._scratch = {}

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, batch: int, pages_per_seq: int, *,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", track: bool = True) -> "PagedKVCache":
        """A cache with zeroed tensors of its own; ``track``: with ``weight`` and ``pos``."""
        device = _cuda(device)
        shape = (num_pages, n_kv_heads, page_size)

        def zeros(*size, dt):
            return torch.zeros(size, dtype=dt, device=device)

        return cls(zeros(*shape, head_dim, dt=dtype), zeros(*shape, head_dim, dt=dtype),
                   zeros(batch, pages_per_seq, dt=torch.int32), zeros(2, batch, dt=torch.int32),
                   weight=zeros(*shape, dt=torch.float32) if track else None,
                   pos=zeros(*shape, dt=torch.int32) if track else None)

    @property
    def lens(self) -> torch.Tensor:
        """Rows held by each sequence (a view of ``counts``)."""
        return self.counts[0]

    def _rows(self, t: torch.Tensor, name: str, heads: Optional[int]):
        """Checks rows of heads; their shape and strides."""
        shape, strides = t.shape, t.stride()
        if len(shape) != 3 or t.dtype != self.dtype or t.get_device() != self._index or shape[2] != self.head_dim or \
                strides[2] != 1 or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {self.head_dim}] "
                             f"{self.dtype} on {self.device}, contiguous in its last dimension")
        return shape, strides

    def _no_gradients(self, tensors, names) -> None:
        """The cache has no derivative: refuses one wanted of an input, or through what is written or read."""
        forward = forward_ad._current_level >= 0
        if forward or torch.is_grad_enabled():
            for t in tensors:
                if t is not None and (forward or t.requires_grad) and _wants_grad(t):
                    name = names[[t is other for other in tensors].index(True)]
                    raise ValueError(f"the cache is not differentiable: {name} needs a gradient (use torch.no_grad())")

    def append(self, k: torch.Tensor, v: torch.Tensor, *, q: Optional[torch.Tensor] = None,
               freqs: Optional[RopeFrequencies] = None, cu_tokens: Optional[torch.Tensor] = None,
               weight: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Writes new rows behind each sequence's last and moves ``counts`` on.

        ``k``, ``v`` ``[tokens, n_kv_heads, head_dim]``, any token and head strides.  One token of each
        sequence (``tokens == batch``), or with ``cu_tokens`` (int32 ``[batch + 1]`` prefix sums
        from 0, on the device) any number of each, none included; tokens behind the last sequence's are
        padding and left out.  With ``freqs``, ``k`` and ``q`` ``[tokens, heads, head_dim]`` are
        rotated to their positions; the rotated ``q`` is returned (rows of padding tokens as they were
        in ``q_out``).  ``weight`` ``[tokens, n_kv_heads]`` fp32 is what the rows start with (0
        otherwise), e.g. what the prompt's own attention gave them.
        """
        (tokens, _, _), (k_token, k_head, _) = self._rows(k, "k", self.n_kv_heads)
        (v_tokens, _, _), (v_token, v_head, _) = self._rows(v, "v", self.n_kv_heads)
        self._no_gradients((k, v, q, q_out, weight, self.k_pages, self.v_pages, self.weight),
                           ("k", "v", "q", "q_out", "weight", "k_pages", "v_pages", "the cache's weight"))
        if v_tokens != tokens:
            raise ValueError(f"k has {tokens} tokens, v has {v_tokens}")
        q_at = q_out_at = q_token = q_head = n_q_heads = rotary = cu_at = weight_at = 0
        written = self._state
        if q is not None:
            (q_tokens, n_q_heads, _), (q_token, q_head, _) = self._rows(q, "q", None)
            if freqs is None:
                raise ValueError("q is only rotated: give freqs, or leave q out")
            if q_tokens != tokens:
                raise ValueError(f"k has {tokens} tokens, q has {q_tokens}")
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.get_device() != self._index or \
                    not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous, of q's shape, type and device")
            else:
                written += (q_out,)
            q_at, q_out_at = q.data_ptr(), q_out.data_ptr()
        if freqs is not None:
            if freqs._index != self._index or freqs.rotary_dim > self.head_dim:
                raise ValueError(f"freqs must be on {self.device} with rotary_dim <= {self.head_dim}")
            rotary = freqs._at
        if cu_tokens is not None:
            if cu_tokens.shape != (self.batch + 1,) or cu_tokens.dtype != torch.int32 or \
                    cu_tokens.get_device() != self._index or not cu_tokens.is_contiguous():
                raise ValueError(f"cu_tokens must be contiguous int32 [{self.batch + 1}] on {self.device}")
            cu_at = cu_tokens.data_ptr()
        elif tokens != self.batch:
            raise ValueError(f"{tokens} tokens for {self.batch} sequences need cu_tokens")
        if weight is not None:
            if self.weight is None or weight.shape != (tokens, self.n_kv_heads) or weight.dtype != torch.float32 or \
                    weight.get_device() != self._index or not weight.is_contiguous():
                raise ValueError(f"weight must be contiguous fp32 [{tokens}, {self.n_kv_heads}] on {self.device}, "
                                 "for a cache that keeps weights")
            weight_at = weight.data_ptr()
        _run("pi05_paged_append", self._index, self._at, _APPEND_ARGS.pack(
            k.data_ptr(), v.data_ptr(), k_token, k_head, v_token, v_head, q_at, q_out_at, q_token, q_head, tokens,
            n_q_heads, cu_at, weight_at, rotary))
        _wrote(written)
        return q_out if q is not None else None

    def attend(self, q: torch.Tensor, *, scale: Optional[float] = None, key_valid: Optional[torch.Tensor] = None,
               track: bool = False, out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of one token of each sequence over its rows: ``q`` ``[batch, heads, head_dim]``
        (any token and head strides), ``heads`` a multiple of ``n_kv_heads``.

        ``scale`` is ``head_dim ** -0.5`` if not given.  ``key_valid`` (bool or uint8 ``[batch, n]``):
        rows that are False are left out, whatever they hold; rows from ``n`` on count (a prompt's
        padding mask need not grow with the sequence).  It speaks of rows, not of positions: once
        :meth:`evict` has moved rows, a mask made before means other tokens, and no one mask can say
        what each head holds.  A cache that evicts is to hold no padding: leave it out of
        :meth:`append` with ``cu_tokens``.  ``track`` adds the probabilities to the
        cache's ``weight`` (its scratch holds a score of every query head for each row that the table
        reaches or, beyond 64 MB, that the pool has).  A sequence with no row gives zeros (lse
        ``-inf``); rows that count but all score ``-inf`` give NaN, as a softmax of them does.
        Returns ``out`` ``[batch, heads, head_dim]``, with ``return_lse`` also the fp32 natural-log
        sums ``[batch, heads]``.
        """
        (batch, heads, dim), (q_token, q_head, _) = self._rows(q, "q", None)
        self._no_gradients((q, out, self.k_pages, self.v_pages, self.weight if track else None),
                           ("q", "out", "k_pages", "v_pages", "the cache's weight"))
        if batch != self.batch or heads == 0 or heads % self.n_kv_heads:
            raise ValueError(f"q must be [{self.batch}, a multiple of {self.n_kv_heads}, {dim}], got {list(q.shape)}")
        if track and self.weight is None:
            raise ValueError("this cache keeps no weights: build it with weight=")
        written = (self.weight,) if track else ()
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != self._index or \
                not out.is_contiguous():
            raise ValueError("out must be contiguous, of q's shape, type and device")
        else:
            written += (out,)
        need, like, like_lse = self._scratch.get((heads, track)) or self._need(heads, track)
        lse = torch.empty_like(like_lse, memory_format=torch.contiguous_format) if return_lse else None
        valid_at = pitch = valid_rows = 0
        if key_valid is not None:
            if key_valid.dim() != 2 or key_valid.dtype not in (torch.bool, torch.uint8) or \
                    key_valid.shape[0] != batch or key_valid.get_device() != self._index or \
                    (key_valid.stride(1) != 1 and key_valid.shape[1] > 1):
                raise ValueError("key_valid must be bool or uint8 [batch, rows] on the cache's device, rows contiguous")
            valid_at, pitch, valid_rows = key_valid.data_ptr(), key_valid.stride(0), key_valid.shape[1]
        # from torch's allocator, call by call: calls on different streams, and graphs, never share it
        scratch = torch.empty_like(like, memory_format=torch.contiguous_format) if need else None
        _run("pi05_paged_attention", self._index, self._at, _ATTEND_ARGS.pack(
            q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), valid_at, q_token, q_head, pitch,
            valid_rows, heads, dim**-0.5 if scale is None else scale, track, scratch.data_ptr() if need else 0, need))
        if written:
            _wrote(written)
        return (out, lse) if return_lse else out

    def _need(self, heads: int, track: bool):
        need = _fn("pi05_paged_attention_scratch_bytes")(self._at, heads, track)
        like = torch.empty(1, dtype=torch.uint8, device=self.device).expand(need)
        like_lse = torch.empty(1, dtype=torch.float32, device=self.device).expand(self.batch, heads)
        self._scratch[heads, track] = need, like, like_lse
        return need, like, like_lse

    def evict(self, budget: int, *, recent: int = 0, sinks: int = 0) -> None:
        """Cuts every sequence with more than ``budget`` rows down to it.

        Each key-value head on its own gives up the rows with the lowest accumulated ``weight``
        (ties: the lowest row first; NaN first of all), those of the ``recent`` newest positions and
        of the first ``sinks`` positions only after all others.  The holes below the budget are filled in
        order by the rows that stay from above it, so the rows of a head are in no order of age
        afterwards: ``pos`` says which token a row is, and a ``key_valid`` made before no longer fits.
        """
        if self.weight is None or self.pos is None:
            raise ValueError("this cache keeps no weights and positions: build it with weight= and pos=")
        if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
            raise ValueError(f"need budget >= 1 and 0 <= recent + sinks <= budget, got {budget}, {recent}, {sinks}")
        self._no_gradients((self.k_pages, self.v_pages, self.weight), ("k_pages", "v_pages", "the cache's weight"))
        if budget >= self.pages_per_seq * self.page_size:
            return  # no sequence can hold more; and below, the numbers fit the library's 32 bits
        _run("pi05_paged_evict", self._index, self._at, budget, recent, sinks)
        _wrote(self._state)

    def read_status(self) -> int:
        """Synchronise, read and clear the cache's device status word (0 = nothing went wrong)."""
        v = ctypes.c_int(0)
        rc = _lib.lib().pi05_read_device_status(self.workspace.data_ptr(), ctypes.byref(v),
                                                torch.cuda.current_stream(self.device).cuda_stream)
        if rc not in (_lib.PI05_OK, 7):
            raise _lib.Pi05Error("pi05_read_device_status", rc, _lib.last_error())
        return v.value
