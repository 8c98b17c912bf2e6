"""Key-value cache, rotary positions and attention: what a language model that
answers over retrieved vectors calls next to the search.

* ``RotaryEmbedding`` -- rotary positions (half or interleaved pairs, part of
  the head, scaled for longer contexts);
* ``PagedKVCache`` -- pages of keys and values resident in HBM, their tables
  and reference counts; ``append``, ``attend``, ``reserve``, ``fork``,
  ``free``, ``compact``, ``copy_pages``; ``share`` finds the prefixes that
  branches share, which ``attend`` then reads once for all of them;
* ``window_attention`` -- causal attention over keys and values as the
  projections left them, through a sliding window with sinks;
* ``cross_attention`` -- attention to keys and values of another length, an
  encoder's states of the documents found.

Tensors are torch tensors on the context's GPU.  Unlike the search calls,
these are queued on torch's current stream and do not wait: a decoder makes
dozens a token.  (Offsets, slots and counts given as host sequences are copied
to the GPU first, which does wait and cannot be captured; int32 tensors there
are used as they are.)  They record no gradients (a tensor that wants one is
refused outside ``torch.no_grad()``, one with a forward-mode tangent always).
They allocate through torch, so a captured graph may hold them.  The reference
keeps its language-model layer on the application's side (LLM/,
Core/ML/Shaders/OptimizedMLShaders.metal:523); there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
import struct

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import VSKError
from .engine import Context

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


# The call's structures as bytes: a decoder makes these calls dozens of times a
# token, and setting a ctypes structure's fields takes several times as long.
# Layouts: vsk_kv, vsk_head_rows, vsk_new_tokens, vsk_attention_args and
# vsk_key_sets of vsk_hip.h.
_KV = struct.Struct("@QQqqqqqqqqQQQQQqiiiiiiii")
_ROWS = struct.Struct("@QQqqqqixxxx")
_NEWS = struct.Struct("@QQiiq")
_ATTEND = struct.Struct("@QQqqqqixxxxQQQqfiii")
_SETS = struct.Struct("@QQqixxxx")
assert _SETS.size == ctypes.sizeof(_lib.vsk_key_sets)
assert _ATTEND.size == ctypes.sizeof(_lib.vsk_attention_args)
assert _KV.size == ctypes.sizeof(_lib.vsk_kv)
assert _ROWS.size == ctypes.sizeof(_lib.vsk_head_rows)
assert _NEWS.size == ctypes.sizeof(_lib.vsk_new_tokens)


def _stream(gpu: int) -> int:
    return torch._C._cuda_getCurrentRawStream(gpu)


def _empty(x):
    """An uninitialised dense tensor like x."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _tensor(gpu, x, name, dtype=None, dims=None):
    """x, checked to be a tensor on that GPU."""
    if not isinstance(x, torch.Tensor) or x.get_device() != gpu:
        raise VSKError(-2, f"{name} must be a tensor on GPU {gpu}, the context's")
    if x.requires_grad and torch.is_grad_enabled():
        # (a result without its history would train on silently)
        raise VSKError(-8, f"{name} requires a gradient, which these calls do not record: detach "
                       "it or call under torch.no_grad()")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise VSKError(-8, f"{name} carries a tangent, which these calls do not pass on")
    if dtype is not None and x.dtype != dtype:
        raise VSKError(-2, f"{name} is {x.dtype}, not {dtype}")
    if dims is not None and x.dim() != dims:
        raise VSKError(-4, f"{name} must have {dims} dimensions, not {x.dim()}")
    return x


def _shared(x):
    """Do tokens or heads of x lie at one place (an expanded tensor)?"""
    (n, h), (a, b) = x.shape[:2], x.stride()[:2]
    return n > 1 and a == 0 or h > 1 and b == 0


def _dense_heads(x):
    """x itself, or a copy whose innermost dimension is dense."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _ints(gpu, x, name):
    """A dense int32 vector on that GPU; a host sequence is copied there."""
    if isinstance(x, torch.Tensor):
        _tensor(gpu, x, name, torch.int32, 1)
        return x if x.is_contiguous() else x.contiguous()
    a = np.asarray(x)
    if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
        raise VSKError(-2, f"{name} must be a vector of whole numbers")
    if a.size and (int(a.min()) < -1 << 31 or int(a.max()) >= 1 << 31):
        raise VSKError(-2, f"{name} does not fit 32 bits")
    return torch.from_numpy(a.astype(np.int32)).to(torch.device("cuda", gpu))


def _rows(src, dst=None):
    x, y = src.stride(), dst.stride() if dst is not None else (0, 0)
    return _ROWS.pack(src.data_ptr(), dst.data_ptr() if dst is not None else 0, x[0], x[1], y[0],
                      y[1], src.shape[1])


class RotaryEmbedding:
    """Rotary positions (``vsk_rotary_*``).

    ``layout``: "half" turns the pairs (i, i + rotary_dim / 2), "interleaved"
    the pairs (2 i, 2 i + 1), of the first ``rotary_dim`` values of a head
    (default: all); the others pass through.  Pair i turns by position *
    base^(-2 i / rotary_dim) radians, changed by ``scaling`` for contexts
    longer than those trained on:

    * ``{"type": "linear", "factor": f}``: positions divided by f;
    * ``{"type": "ntk", "factor": f}``: base * f^(r / (r - 2)), which leaves
      the fastest pair as it is and divides the slowest one's by f;
    * ``{"type": "yarn", "factor": f, "original_length": n}``: pairs that turn
      more than ``beta_fast`` (32) times over n positions stay, those under
      ``beta_slow`` (1) are divided by f, those between are blended, and the
      rotated values are multiplied by ``attention_factor``
      (0.1 ln f + 1);
    * ``{"type": "given", "inv_freq": x}``: the pairs' radians a position
      themselves (``rotary_dim / 2`` of them, whatever the base), and an
      ``attention_factor`` (1)."""

    LAYOUTS = {"half": 0, "interleaved": 1}

    def __init__(self, ctx: Context, head_dim: int, rotary_dim: int | None = None,
                 base: float = 10000.0, layout: str = "half", scaling: dict | None = None):
        r = head_dim if rotary_dim is None else int(rotary_dim)
        if layout not in self.LAYOUTS:
            raise VSKError(-2, f"unknown rotary layout {layout!r}")
        if r < 2 or r % 2 or r > head_dim:
            raise VSKError(-2, "rotary_dim must be even, at least 2 and at most head_dim")
        if not base > 0:
            raise VSKError(-2, "base must be positive")
        self.ctx, self.head_dim, self.rotary_dim, self.layout = ctx, int(head_dim), r, layout
        self.inv_freq, self.amplitude = self.frequencies(r, base, scaling)
        f = np.ascontiguousarray(self.inv_freq, np.float64)
        h = ctypes.c_void_p()
        ctx.check(ctx.lib.vsk_rotary_create(ctx.handle, f.ctypes.data, r // 2,
                                            self.LAYOUTS[layout], self.amplitude,
                                            ctypes.byref(h)))
        self.handle = h

    @staticmethod
    def frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None):
        """(radians a position for each pair, factor on the rotated values)."""
        r = rotary_dim
        i = np.arange(r // 2, dtype=np.float64)
        inv = float(base) ** (-2.0 * i / r)
        if not scaling:
            return inv, 1.0
        s = dict(scaling)
        kind, amplitude = s.pop("type", None), 1.0
        if kind == "given":
            given = s.pop("inv_freq", None)
            inv = np.array(() if given is None else given, np.float64)
            if inv.shape != (r // 2,):
                raise VSKError(-2, f"inv_freq must hold a value for each of {r // 2} pairs")
            amplitude = float(s.pop("attention_factor", 1.0))
            if s:
                raise VSKError(-2, f"unknown scaling options {sorted(s)}")
            return inv, amplitude
        f = float(s.pop("factor", 0))
        if not f >= 1:
            raise VSKError(-2, "scaling needs a factor of at least 1")
        if kind == "linear":
            inv = inv / f
        elif kind == "ntk":
            if r < 4:
                raise VSKError(-2, "ntk scaling needs two pairs at least")
            inv = (base * f ** (r / (r - 2.0))) ** (-2.0 * i / r)
        elif kind == "yarn":
            n = float(s.pop("original_length", 0))
            fast, slow = float(s.pop("beta_fast", 32.0)), float(s.pop("beta_slow", 1.0))
            if not n > 0 or not fast > slow > 0 or not base > 1:
                raise VSKError(-2, "yarn scaling needs original_length, beta_fast > beta_slow > 0 "
                               "and a base over 1")

            def pair(turns):  # the pair that turns so often over n positions
                return r * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))

            low = max(math.floor(pair(fast)), 0)
            high = min(math.ceil(pair(slow)), r - 1)
            ramp = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
            inv = inv * (1 - ramp) + inv / f * ramp
            amplitude = float(s.pop("attention_factor", 0.1 * math.log(f) + 1.0))
        else:
            raise VSKError(-2, f"unknown scaling {kind!r}")
        if s:
            raise VSKError(-2, f"unknown scaling options {sorted(s)}")
        return inv, amplitude

    def free(self):
        if getattr(self, "handle", None):
            self.ctx.lib.vsk_rotary_free(self.ctx.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def apply(self, q, k=None, *, positions, inverse: bool = False, inplace: bool = False):
        """q (and k), tokens x heads x head_dim, turned by positions (int32,
        one a token): new tensors, or the given ones with ``inplace``.
        ``inverse`` turns back, with the same factor on the rotated values:
        the gradient of ``apply``.  With positions p - p' it moves a cached
        key from p to p', times that factor (``amplitude``): divide by it where
        it is not 1 (yarn)."""
        ctx, gpu = self.ctx, self.ctx.device
        tokens, dtype = self._checked(_tensor(gpu, q, "q", None, 3), "q", None), q.dtype
        if k is not None:
            self._checked(_tensor(gpu, k, "k", dtype, 3), "k", tokens)
        if dtype not in _TYPES:
            raise VSKError(-8, f"{dtype} is not supported")
        if _tensor(gpu, positions, "positions", torch.int32, 1).shape[0] != tokens:
            raise VSKError(-4, f"{positions.shape[0]} positions for {tokens} tokens")
        positions = positions.contiguous()
        if inplace:
            if q.stride(-1) != 1 or k is not None and k.stride(-1) != 1:
                raise VSKError(-2, "inplace needs dense heads")
            if _shared(q) or k is not None and _shared(k):
                # (threads would turn what others have turned already)
                raise VSKError(-2, "inplace needs tokens and heads with memory of their own")
            to_q, to_k = q, k
        else:
            q = _dense_heads(q)
            to_q, to_k = _empty(q), None
            if k is not None:
                k = _dense_heads(k)
                to_k = _empty(k)
        rows = _rows(q, to_q) if q.shape[1] else b""
        if k is not None and k.shape[1]:
            rows += _rows(k, to_k)
        if tokens and rows:
            status = ctx.lib.vsk_rotary_apply(
                ctx.handle, _stream(gpu), self.handle, _TYPES[dtype], self.head_dim, tokens,
                positions.data_ptr(), 1 if inverse else 0, rows, len(rows) // _ROWS.size)
            if status:
                ctx.check(status)
        return to_q if k is None else (to_q, to_k)

    def _checked(self, x, name, tokens):
        n, _, d = x.shape
        if d != self.head_dim or tokens is not None and n != tokens:
            raise VSKError(-4, f"{name} is {tuple(x.shape)}: head_dim is {self.head_dim}"
                           + (f", tokens are {tokens}" if tokens is not None else ""))
        return n


def _attend(ctx, kv, layer, q, news, k_starts, scale, window, sinks, max_length, return_lse,
            sets=None, shared=None):
    """The checked call of vsk_attention (``sets``: vsk_cross_attention,
    ``shared``: vsk_attention_shared)."""
    if window is not None and window < 1:
        raise VSKError(-2, "window must be at least 1 (None: no window)")
    if sinks < 0:
        raise VSKError(-2, "sinks must not be negative")
    out, x = _empty(q), q.stride()
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    heads, y = q.shape[1], out.stride()
    lib, handle, work, need = ctx.lib, ctx.handle, None, 0
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    window, max_length = window or 0, max_length or 0
    if max(window, sinks, max_length) >= 1 << 31:
        raise VSKError(-9, "window, sinks and max_length are 32-bit")
    while True:
        a = _ATTEND.pack(q.data_ptr(), out.data_ptr(), x[0], x[1], y[0], y[1], heads,
                         lse.data_ptr() if return_lse else 0, k_starts,
                         work.data_ptr() if need else 0, need,
                         scale, window, sinks, max_length)
        if need:
            break
        if sets is not None:
            need = lib.vsk_cross_attention_workspace(handle, kv, news, a)
        elif shared is not None:
            need = lib.vsk_attention_shared_workspace(handle, kv, news, a, shared)
        else:
            need = lib.vsk_attention_workspace(handle, kv, news, a)
        if not need:
            break
        work = torch.empty(need, dtype=torch.uint8, device=q.device)
    stream = _stream(ctx.device)
    if sets is not None:
        status = lib.vsk_cross_attention(handle, stream, kv, news, a, sets)
    elif shared is not None:
        status = lib.vsk_attention_shared(handle, stream, kv, layer, news, a, shared)
    else:
        status = lib.vsk_attention(handle, stream, kv, layer, news, a)
    if status:
        ctx.check(status)
    return (out, lse) if return_lse else out


class PagedKVCache:
    """Keys and values of many sequences in pages of ``page_size`` tokens (a
    power of two, at least 16).

    ``k``, ``v``: layers x pages x page_size x kv_heads x head_dim;
    ``table`` (int32, slots x width): the pages of the sequence in each slot,
    -1 where there is none; ``lengths`` (int32, slots); ``refs`` (int32,
    pages): how many sequences hold a page.  A page that is full may be
    shared; one that is not belongs to one sequence.

    A step of a decoder: ``reserve`` makes room for the new tokens, then each
    layer calls ``append`` with their keys and values and ``attend`` with
    their queries.  New tokens are always a sequence's last ones."""

    def __init__(self, ctx: Context, *, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 slots: int, width: int, layers: int = 1, dtype=torch.bfloat16):
        for name, x in (("pages", pages), ("kv_heads", kv_heads), ("head_dim", head_dim),
                        ("slots", slots), ("width", width), ("layers", layers)):
            if x < 1:
                raise VSKError(-2, f"{name} must be positive")
        dev = torch.device("cuda", ctx.device)
        shape = (layers, pages, page_size, kv_heads, head_dim)
        if dtype not in _TYPES:
            raise VSKError(-8, f"{dtype} is not supported")
        k, v = (torch.empty(shape, dtype=dtype, device=dev) for _ in range(2))
        table = torch.full((slots, width), -1, dtype=torch.int32, device=dev)
        self._hold(ctx, k, v, table, torch.zeros(slots, dtype=torch.int32, device=dev),
                   torch.zeros(pages, dtype=torch.int32, device=dev))

    @classmethod
    def over(cls, ctx: Context, k, v, table, lengths, refs=None) -> "PagedKVCache":
        """A cache over tensors that the caller holds (k and v may lack the
        layers' dimension, and may have any strides over dense heads).
        Without ``refs`` there is no page keeping, only ``append`` and
        ``attend``."""
        self = cls.__new__(cls)
        self._hold(ctx, k, v, table, lengths, refs)
        return self

    def _hold(self, ctx, k, v, table, lengths, refs):
        for x, name in ((k, "k"), (v, "v")):
            _tensor(ctx.device, x, name)
            if x.dim() not in (4, 5):
                raise VSKError(-4, f"{name} must be (layers x) pages x page_size x kv_heads x "
                               "head_dim")
            if x.dtype not in _TYPES:
                raise VSKError(-8, f"{x.dtype} is not supported")
            if x.stride(-1) != 1 and x.shape[-1] != 1:
                raise VSKError(-2, f"the heads of {name} must be dense")
        if k.shape != v.shape or k.dtype != v.dtype:
            raise VSKError(-4, "k and v differ in shape or type")
        _tensor(ctx.device, table, "table", torch.int32, 2)
        _tensor(ctx.device, lengths, "lengths", torch.int32, 1)
        if table.shape[0] != lengths.shape[0] or table.stride(1) != 1 and table.shape[1] != 1:
            raise VSKError(-4, "table must be slots x width, dense rows, lengths of slots")
        if lengths.stride(0) != 1 and lengths.shape[0] != 1:
            raise VSKError(-2, "lengths must be dense")
        k5, v5 = (x if x.dim() == 5 else x[None] for x in (k, v))
        layers, pages, page_size, kv_heads, head_dim = k5.shape
        if max(layers, pages, kv_heads, *table.shape) >= 1 << 31:
            raise VSKError(-9, "the cache's counts are 32-bit")
        if page_size < 16 or page_size & (page_size - 1):
            raise VSKError(-8, "page_size must be a power of two of at least 16")
        self.ctx, self.k, self.v = ctx, k, v
        self.table, self.lengths, self.refs = table, lengths, refs
        self.layers, self.pages, self.page_size = layers, pages, page_size
        self.kv_heads, self.head_dim, self.dtype = kv_heads, head_dim, k.dtype
        self.slots, self.width = table.shape
        self.device, self.gpu = k.device, ctx.device
        kv = _lib.vsk_kv()
        kv.k, kv.v = k.data_ptr(), v.data_ptr()
        kv.k_layer, kv.k_page, kv.k_row, kv.k_head = k5.stride()[:4]
        kv.v_layer, kv.v_page, kv.v_row, kv.v_head = v5.stride()[:4]
        kv.table, kv.lengths = table.data_ptr(), lengths.data_ptr()
        kv.table_stride = table.stride(0)
        kv.dtype, kv.layers, kv.pages, kv.page_size = _TYPES[k.dtype], layers, pages, page_size
        kv.kv_heads, kv.head_dim, kv.slots, kv.width = kv_heads, head_dim, self.slots, self.width
        if refs is not None:
            _tensor(ctx.device, refs, "refs", torch.int32, 1)
            if refs.shape[0] != pages or refs.stride(0) != 1 and pages != 1:
                raise VSKError(-4, "refs must be a dense vector of a count a page")
            self.status = torch.zeros(4, dtype=torch.int32, device=k.device)
            self._scratch = torch.empty(ctx.lib.vsk_kv_scratch_ints(pages, self.slots),
                                        dtype=torch.int32, device=k.device)
            kv.refs, kv.status = refs.data_ptr(), self.status.data_ptr()
            kv.scratch = self._scratch.data_ptr()
        self._kv = kv
        self._ref = ctypes.byref(kv)

    # -- new tokens -----------------------------------------------------------
    def _layer(self, layer):
        if not 0 <= layer < self.layers:  # (the call would take its low 32 bits)
            raise VSKError(-2, f"no layer {layer}: the cache has {self.layers}")

    def _news(self, x, starts, seqs, max_new):
        """vsk_new_tokens of the rows of x and what must outlive the call."""
        tokens = x.shape[0]
        n, most, at = tokens, 1, None
        if starts is not None:
            at = _ints(self.gpu, starts, "starts")
            n = at.shape[0] - 1
            if n < 0:
                raise VSKError(-4, "starts holds an offset a sequence and the end")
            most = tokens if max_new is None else min(int(max_new), tokens)
            if most < 0:
                raise VSKError(-2, "max_new must not be negative")
        if seqs is not None:
            seqs = _ints(self.gpu, seqs, "seqs")
            if seqs.shape[0] != n:
                raise VSKError(-4, f"{seqs.shape[0]} slots for {n} sequences")
        elif n > self.slots:
            raise VSKError(-2, f"{n} sequences, {self.slots} slots")
        return _NEWS.pack(at.data_ptr() if at is not None else 0,
                          seqs.data_ptr() if seqs is not None else 0, n, most, tokens), (at, seqs)

    def _heads(self, x, name, heads=None):
        _tensor(self.gpu, x, name, self.dtype, 3)
        if x.shape[2] != self.head_dim or heads is not None and x.shape[1] != heads:
            raise VSKError(-4, f"{name} is {tuple(x.shape)}: heads of {self.head_dim} are wanted"
                           + (f", {heads} of them" if heads is not None else ""))
        return _dense_heads(x)

    def append(self, k, v, *, starts=None, seqs=None, max_new=None, layer: int = 0,
               rotary: RotaryEmbedding | None = None, q=None):
        """Writes the new tokens' keys and values (tokens x kv_heads x
        head_dim) to their places.  Sequence i, in slot ``seqs[i]`` (default:
        i), has the rows ``starts[i] .. starts[i + 1]`` (default: row i); they
        are the last of its length.  No sequence has more than ``max_new``
        (default: all the rows; the nearer the bound, the fewer blocks start
        for nothing).  ``rotary`` turns the keys by their positions, and ``q``,
        returned turned, with them.  Rows of no sequence, and a sequence's
        past ``max_new``, are not treated: what is returned for them is
        undefined."""
        self._layer(layer)
        k, v = self._heads(k, "k", self.kv_heads), self._heads(v, "v", self.kv_heads)
        if v.shape[0] != k.shape[0]:
            raise VSKError(-4, f"{k.shape[0]} keys, {v.shape[0]} values")
        if rotary is not None:
            if not rotary.handle:
                raise VSKError(-2, "the rotary embedding has been freed")
            if rotary.head_dim != self.head_dim:
                raise VSKError(-4, f"rotary is for heads of {rotary.head_dim}")
        news, keep = self._news(k, starts, seqs, max_new)
        out, qr = None, None
        if q is not None:
            q = self._heads(q, "q")
            if q.shape[0] != k.shape[0]:
                raise VSKError(-4, f"{k.shape[0]} keys, {q.shape[0]} queries")
            out = _empty(q)
            qr = _rows(q, out)
        if k.shape[0]:
            self.ctx.check(self.ctx.lib.vsk_kv_append(
                self.ctx.handle, _stream(self.gpu), self._ref, layer, news, _rows(k), _rows(v),
                rotary.handle if rotary is not None else None, qr))
        return out

    def attend(self, q, *, starts=None, seqs=None, max_new=None, layer: int = 0,
               scale: float | None = None, window: int | None = None, sinks: int = 0,
               max_length: int | None = None, return_lse: bool = False,
               shared: "SharedPrefix | None" = None):
        """Attention of the new tokens' queries (tokens x heads x head_dim;
        consecutive heads share a key head) over their sequences in the
        cache, laid out as in ``append``.  A token sees the keys up to its own
        position, with a ``window`` only the last ``window`` of them and the
        first ``sinks``.  ``scale`` defaults to head_dim^-0.5; ``max_length``
        bounds the lengths, to divide the work by (default: the table's
        width).  Returns the outputs, with ``return_lse`` also the logarithm
        of each row's sum (-inf, and zeros, where a row sees nothing; undefined
        for rows that are not treated).

        Scores, sums and outputs are computed in 32 bits.  In 16 bits a weight
        is rounded before it multiplies a value: for few rows to two 16-bit
        parts, for many (prompts) once to the values' type, which is off by as
        much as the output's own rounding.

        ``shared``, of ``share``: the same attention, in which the keys that a
        group of sequences shares are read once for all of them.  Its
        sequences, or the first of them, are the call's (``seqs`` is not given
        again).  Where a sequence has more than ``max_new`` tokens the results
        of its whole group are undefined.  A group's rows count together as few
        or many: a prefix that many branches share rounds its weights once, as
        a prompt does, also for one token of each.  With a window each sequence
        reads its own keys."""
        self._layer(layer)
        q = self._heads(q, "q")
        if shared is not None:
            if not isinstance(shared, SharedPrefix) or shared.cache is not self:
                raise VSKError(-2, "shared must be what this cache's share() returned")
            if seqs is not None:
                raise VSKError(-2, "the slots are those that share() was called with")
            if starts is not None:
                starts = _ints(self.gpu, starts, "starts")
            n = q.shape[0] if starts is None else max(starts.shape[0] - 1, 0)
            if n > shared.n:
                raise VSKError(-4, f"{n} sequences, share() knows {shared.n}")
            seqs = shared.seqs if shared.seqs is None or n == shared.n else shared.seqs[:n]
            shared = shared._ref
        if q.shape[1] % self.kv_heads or not q.shape[1]:
            raise VSKError(-4, f"{q.shape[1]} query heads over {self.kv_heads} key heads")
        news, keep = self._news(q, starts, seqs, max_new)
        return _attend(self.ctx, self._ref, layer, q, news, 0, scale, window, sinks, max_length,
                       return_lse, None, shared)

    def share(self, groups, *, seqs=None, members: int | None = None,
              prefix: int | None = None) -> "SharedPrefix":
        """Finds the pages that groups of sequences share, for ``attend``:
        group g are the sequences ``groups[g] .. groups[g + 1]`` (ascending
        offsets) of those in slots ``seqs`` (default: slot i is sequence i).
        Nothing is assumed of them: a group's prefix is the leading whole pages
        that all its members' tables agree on (one alone has all its own).
        What is found stays true while the sequences grow and the pool is
        compacted, also where one has been cut back since (its length lowered).
        Call ``update`` of what is returned after a ``fork`` into, or a ``free``
        of, one of these slots, and after a sequence that was cut back into its
        prefix has grown again (``reserve`` gives it pages of its own there: its
        group would read pages that are not theirs).
        Sharing pays from contexts of some thousand keys on: a second launch
        joins the parts (4 branches of 512 keys take 13 us with it and
        10 without, 8 of 8,192 18 and 30, 64 of 32,768 76 and 411: 32 heads
        of 128 on 8).
        ``members`` bounds a group's sequences (default: known of a host
        sequence, all of them otherwise; a group of more shares nothing),
        ``prefix`` says about how many keys the longest prefix has, to divide
        the work by: a sequence with more keys of its own than are left of
        ``max_length`` then is better in a group, alone if need be, than in
        none."""
        return SharedPrefix(self, groups, seqs, members, prefix)

    # -- pages ------------------------------------------------------------------
    def _keeping(self):
        if self.refs is None:
            raise VSKError(-8, "a cache without refs keeps no pages")

    def _known(self, x, name, distinct=False):
        """Checks slots that are known on the host (those on the GPU are the
        caller's to keep in range and distinct)."""
        if isinstance(x, torch.Tensor):
            return
        a = np.asarray(x)
        if a.size and (a.min() < 0 or a.max() >= self.slots):
            raise VSKError(-2, f"{name} outside the {self.slots} slots")
        if distinct and np.unique(a).size != a.size:
            raise VSKError(-2, f"{name} must be distinct")

    def reserve(self, seqs, counts):
        """Grows the sequences in these slots (distinct) by these numbers of
        tokens, taking the lowest free pages; ``missing()`` tells of a
        shortage.  A sequence may be cut back first, by a lower length in
        ``lengths`` (whole pages, where its pages are shared): new pages take
        the place of those that it held past that."""
        self._keeping()
        self._known(seqs, "seqs", distinct=True)
        s, c = _ints(self.gpu, seqs, "seqs"), _ints(self.gpu, counts, "counts")
        if s.shape != c.shape:
            raise VSKError(-4, f"{s.shape[0]} slots, {c.shape[0]} counts")
        self.ctx.check(self.ctx.lib.vsk_kv_reserve(self.ctx.handle, _stream(self.gpu),
                                                   self._ref, s.data_ptr(), c.data_ptr(),
                                                   s.shape[0]))

    def fork(self, parents, children):
        """The sequences in slots ``children`` become branches of those in
        ``parents``: whole pages are shared, a last page that is not full is
        copied; ``missing()`` tells of children that found none for it, which
        keep the whole pages only.  What the children held is released."""
        self._keeping()
        self._known(parents, "parents")
        self._known(children, "children", distinct=True)
        if not isinstance(parents, torch.Tensor) and not isinstance(children, torch.Tensor):
            if set(children) & set(parents):
                raise VSKError(-2, "a child must not be a parent")
        p, c = _ints(self.gpu, parents, "parents"), _ints(self.gpu, children, "children")
        if p.shape != c.shape:
            raise VSKError(-4, f"{p.shape[0]} parents, {c.shape[0]} children")
        self.ctx.check(self.ctx.lib.vsk_kv_fork(self.ctx.handle, _stream(self.gpu), self._ref,
                                                p.data_ptr(), c.data_ptr(), p.shape[0]))

    def free(self, seqs):
        """Releases the pages of the sequences in these slots."""
        self._keeping()
        self._known(seqs, "seqs")
        s = _ints(self.gpu, seqs, "seqs")
        self.ctx.check(self.ctx.lib.vsk_kv_free(self.ctx.handle, _stream(self.gpu), self._ref,
                                                s.data_ptr(), s.shape[0]))

    def compact(self):
        """Moves the pages in use to the low end of the pool, as few as that
        takes; returns their number (an int32 tensor, the cache's own)."""
        self._keeping()
        self.ctx.check(self.ctx.lib.vsk_kv_compact(self.ctx.handle, _stream(self.gpu),
                                                   self._ref))
        return self.status[1]

    def copy_pages(self, src, dst):
        """Copies pages ``src`` to pages ``dst`` in every layer.  No page may be
        written twice, or be both read and written."""
        self._keeping()
        s, d = _ints(self.gpu, src, "src"), _ints(self.gpu, dst, "dst")
        if s.shape != d.shape:
            raise VSKError(-4, f"{s.shape[0]} sources, {d.shape[0]} destinations")
        self.ctx.check(self.ctx.lib.vsk_kv_copy(self.ctx.handle, _stream(self.gpu), self._ref,
                                                s.data_ptr(), d.data_ptr(), s.shape[0]))

    def missing(self) -> int:
        """Pages that the last ``reserve`` or ``fork`` found none for (waits
        for the stream)."""
        self._keeping()
        return int(self.status[0])


class SharedPrefix:
    """What ``PagedKVCache.share`` found: ``prefix``, the keys that each
    sequence's group shares (int32, on the GPU)."""

    def __init__(self, cache: PagedKVCache, groups, seqs, members, prefix):
        gpu = cache.gpu
        self.cache = cache
        self.seqs = None if seqs is None else _ints(gpu, seqs, "seqs")
        if seqs is not None:
            cache._known(seqs, "seqs")
        self.n = cache.slots if seqs is None else self.seqs.shape[0]
        if not isinstance(groups, torch.Tensor):
            a = np.asarray(groups)
            if a.ndim != 1 or a.size < 1 or a.dtype.kind not in "iu":
                raise VSKError(-2, "groups holds an offset a group and the end")
            if a.min() < 0 or a.max() > self.n or (a[1:] < a[:-1]).any():
                raise VSKError(-2, f"groups must ascend from 0 to at most {self.n}")
            known = int((a[1:] - a[:-1]).max()) if a.size > 1 else 0
            members = known if members is None or 0 <= members < known else members
        self.groups = _ints(gpu, groups, "groups")
        if self.groups.shape[0] < 1:
            raise VSKError(-2, "groups holds an offset a group and the end")
        members = self.n if members is None else min(int(members), self.n)
        most = 0 if prefix is None else int(prefix)
        if members < 0 or not 0 <= most < 1 << 31:
            raise VSKError(-2, "members and prefix are counts")
        self.prefix = torch.zeros(self.n, dtype=torch.int32, device=cache.device)
        self._c = _lib.vsk_shared_prefix(self.groups.data_ptr(), self.prefix.data_ptr(),
                                         self.groups.shape[0] - 1, self.n, members, most)
        self._ref = ctypes.byref(self._c)
        self.update()

    def update(self):
        """Finds the prefixes anew, in the same tensors."""
        c = self.cache
        c.ctx.check(c.ctx.lib.vsk_kv_share(c.ctx.handle, _stream(c.gpu), c._ref,
                                           self.seqs.data_ptr() if self.seqs is not None else None,
                                           self._ref))


def cross_attention(ctx: Context, q, k, v, *, starts=None, k_starts=None, k_lengths=None,
                    sets=None, max_length: int | None = None, max_keys: int | None = None,
                    scale: float | None = None, return_lse: bool = False):
    """Attention to keys and values of another length, all of which every query
    sees: a decoder's tokens to an encoder's states of the documents found.

    q is tokens x heads x head_dim; sequence i its rows ``starts[i] ..
    starts[i + 1]`` (default: row i alone, a decoding step's).  k and v are
    rows x kv_heads x head_dim with ``k_starts``, the offsets of the sets of
    keys (and the end), or a padded batch, sets x length x kv_heads x head_dim,
    with ``k_lengths`` (default: all of them are keys).  Sequence i sees set
    ``sets[i]`` (default: i); several may see one (tokens side by side that do
    are fastest as one sequence), and one that is not there (-1) is empty. A
    query that sees no key gets zeros (and -inf). ``max_length`` bounds a
    sequence's queries, ``max_keys`` a set's keys, to divide the work by
    (default: all rows, or the padded length). scale, return_lse, the rounding
    of weights and the rows that are not treated as in ``PagedKVCache.attend``;
    keys past a set's length may hold anything."""
    gpu = ctx.device
    dtype = _tensor(gpu, q, "q", None, 3).dtype
    _tensor(gpu, k, "k", dtype), _tensor(gpu, v, "v", dtype)
    if dtype not in _TYPES:
        raise VSKError(-8, f"{dtype} is not supported")
    if k.shape != v.shape or k.dim() not in (3, 4) or q.shape[2] != k.shape[-1]:
        raise VSKError(-4, f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    tokens, heads, d = q.shape
    kv_heads = k.shape[-2]
    if not heads or not kv_heads or heads % kv_heads:
        raise VSKError(-4, f"{heads} query heads over {kv_heads} key heads")
    q, k, v = _dense_heads(q), _dense_heads(k), _dense_heads(v)
    at = lengths = None
    step = 0
    if k.dim() == 3:
        if k_starts is None or k_lengths is not None:
            raise VSKError(-2, "rows of keys take k_starts, a padded batch k_lengths")
        at = _ints(gpu, k_starts, "k_starts")
        if at.shape[0] < 1:
            raise VSKError(-4, "k_starts holds an offset a set and the end")
        n_sets, rows = at.shape[0] - 1, k.shape[0]
        x, y = k.stride(), v.stride()
    else:
        if k_starts is not None:
            raise VSKError(-2, "rows of keys take k_starts, a padded batch k_lengths")
        n_sets, rows = k.shape[:2]
        if k_lengths is not None:
            lengths = _ints(gpu, k_lengths, "k_lengths")
            if lengths.shape[0] != n_sets:
                raise VSKError(-4, f"{lengths.shape[0]} lengths for {n_sets} sets")
        (k, x, step), (v, y, other) = _padded(k), _padded(v)
        if step != other:
            (k, x, step), (v, y, _) = _padded(k.contiguous()), _padded(v.contiguous())
    if max(rows, kv_heads, heads, step) > 1 << 30 or n_sets >= 1 << 31:
        raise VSKError(-9, f"{rows} keys of {kv_heads} heads: at most 2^30")
    n, most, s = tokens, 1, None
    if starts is not None:
        s = _ints(gpu, starts, "starts")
        n = s.shape[0] - 1
        if n < 0:
            raise VSKError(-4, "starts holds an offset a sequence and the end")
        most = tokens if max_length is None else min(int(max_length), tokens)
        if most < 0:
            raise VSKError(-2, "max_length must not be negative")
    which = None
    if sets is not None:
        which = _ints(gpu, sets, "sets")
        if which.shape[0] != n:
            raise VSKError(-4, f"{which.shape[0]} sets for {n} sequences")
    elif n > n_sets:
        raise VSKError(-4, f"{n} sequences, {n_sets} sets of keys")
    if not rows or not n_sets:
        # (no memory that could be read: one empty set)
        k, v, x, y, step, rows = q, q, (q.stride(0), 0), (q.stride(0), 0), 0, 0
        at, lengths, n_sets, which = None, None, 1, torch.zeros_like(
            which) if which is not None else torch.zeros(n, dtype=torch.int32, device=q.device)
    kv = _KV.pack(k.data_ptr(), v.data_ptr(), 0, 0, x[0], x[1], 0, 0, y[0], y[1], 0, 0, 0, 0, 0,
                  0, _TYPES[dtype], 1, rows, 0, kv_heads, d, 0, 0)
    news = _NEWS.pack(s.data_ptr() if s is not None else 0,
                      which.data_ptr() if which is not None else 0, n, most, tokens)
    key_sets = _SETS.pack(at.data_ptr() if at is not None else 0,
                          lengths.data_ptr() if lengths is not None else 0, step, n_sets)
    return _attend(ctx, kv, 0, q, news, 0, scale, None, 0, max_keys, return_lse, key_sets)


def _padded(x):
    """x, sets x length x heads x d, its row and head strides, and the rows
    from a set to the next (x, or a copy where that is no whole number)."""
    a, b, c = x.stride()[:3]
    if x.shape[0] <= 1:
        return x, (b, c), x.shape[1]
    if x.shape[1] <= 1 and 0 < a <= 1 << 26:
        return x, (a, c), 1  # (the stride between a set's rows may be any)
    if b <= 0 or a % b:
        x = x.contiguous()
        a, b, c = x.stride()[:3]
    return x, (b, c), a // b


def window_attention(ctx: Context, q, k, v, *, starts, k_starts=None, max_length: int | None = None,
                     max_keys: int | None = None, scale: float | None = None,
                     window: int | None = None, sinks: int = 0, return_lse: bool = False):
    """Causal attention of ragged sequences over dense keys and values: q is
    tokens x heads x head_dim, sequence i its rows ``starts[i] ..
    starts[i + 1]``; k and v are rows x kv_heads x head_dim with the offsets
    ``k_starts`` (default: ``starts``), the queries standing at the keys' end.
    ``max_length`` bounds the sequences' queries (default: all rows),
    ``max_keys`` their keys, to divide the work by (default: ``max_length``
    without ``k_starts``, else all rows); window,
    sinks, scale, return_lse, the rounding of weights and the rows that are not
    treated as in ``PagedKVCache.attend``."""
    gpu = ctx.device
    dtype = _tensor(gpu, q, "q", None, 3).dtype
    _tensor(gpu, k, "k", dtype, 3), _tensor(gpu, v, "v", dtype, 3)
    if q.dtype not in _TYPES:
        raise VSKError(-8, f"{q.dtype} is not supported")
    if k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise VSKError(-4, f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if not q.shape[1] or not k.shape[1] or q.shape[1] % k.shape[1]:
        raise VSKError(-4, f"{q.shape[1]} query heads over {k.shape[1]} key heads")
    if not k.shape[0] and q.shape[0]:
        raise VSKError(-3, "no keys")
    q, k, v = _dense_heads(q), _dense_heads(k), _dense_heads(v)
    s = _ints(gpu, starts, "starts")
    ks = s if k_starts is None else _ints(gpu, k_starts, "k_starts")
    if s.shape[0] < 1 or ks.shape != s.shape:
        raise VSKError(-4, "starts and k_starts hold an offset a sequence and the end")
    if k_starts is None and k.shape[0] != q.shape[0]:
        raise VSKError(-4, f"{q.shape[0]} queries, {k.shape[0]} keys: k_starts is wanted")
    rows, heads, d = k.shape
    if max(rows, heads, q.shape[1]) > 1 << 30:
        raise VSKError(-9, f"{rows} keys of {heads} heads: at most 2^30")
    x, y = k.stride(), v.stride()
    # (dense rows: no table, no pages, no layers but one)
    kv = _KV.pack(k.data_ptr(), v.data_ptr(), 0, 0, x[0], x[1], 0, 0, y[0], y[1], 0, 0, 0, 0, 0,
                  0, _TYPES[dtype], 1, rows, 0, heads, d, 0, 0)
    most = q.shape[0] if max_length is None else min(int(max_length), q.shape[0])
    news = _NEWS.pack(s.data_ptr(), 0, s.shape[0] - 1, most, q.shape[0])
    if max_keys is None and k_starts is None:
        max_keys = max_length
    return _attend(ctx, kv, 0, q, news, ks.data_ptr(), scale, window, sinks, max_keys, return_lse)
