"""Operators behind a prompt on torch tensors: positions by rotation, a key/value cache of pages,
attention of new tokens over it.  The thin mirror of the mononn_rotary_* and mononn_paged_* part of
include/mononn.h; the reference has no counterpart (its decoder graphs end with the prompt).

Each operator comes as a function, and as a runner (`rotary_runner`, `PagedCache.append_runner`,
`PagedCache.attention_runner`): the arguments are checked and their addresses and sizes taken once, and
the returned zero-argument callable does nothing but the library call (and tells autograd what was
written), for serving loops that reuse their buffers (what page tables, lengths, indptr and positions
hold is read on the device at each call).  A runner keeps its tensors alive; its stream is the one
given, or torch's current stream of the tensors' device when it was made.
"""
from __future__ import annotations

import ctypes as C
import dataclasses
import functools

from . import capi
from .capi import check, lib

_SCALINGS = {"none": 0, "linear": 1, "base": 2, "ramp": 3, "bands": 4}


@dataclasses.dataclass(frozen=True)
class Rotary:
    """A rotary embedding: which elements of a head turn, in which pairs, and how fast (the scalings are
    those of mononn_rotary_config; None or 0 stands for the default)."""
    rotary_dim: int
    interleaved: bool = False
    theta: float | None = 10000.0
    scaling: str = "none"  # none, linear, base, ramp, bands
    factor: float | None = 1.0           # has no default where a scaling uses it
    original_length: float | None = 0.0  # has none, either
    low: float | None = 0.0
    high: float | None = 0.0
    magnitude: float | None = 0.0

    def table(self) -> capi.RotaryTable:
        """Turning rates (shares of a full turn per position) as the kernels take them."""
        if self.scaling not in _SCALINGS:
            raise ValueError(f"scaling must be one of {sorted(_SCALINGS)}")
        if not 0 <= self.rotary_dim < 2**32:
            raise ValueError("rotary_dim out of range")
        c = capi.RotaryConfigArgs(self.rotary_dim, int(self.interleaved), _SCALINGS[self.scaling], *(
            0.0 if x is None else x
            for x in (self.theta, self.factor, self.original_length, self.low, self.high, self.magnitude)))
        t = capi.RotaryTable()
        check(lib().mononn_rotary_init(C.byref(c), C.byref(t)))
        return t


def _dtype(t) -> int:
    import torch
    if t.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"float16 or bfloat16 tensors are needed, not {t.dtype}")
    return int(t.dtype == torch.bfloat16)


@functools.cache
def _autograd():
    import torch
    return torch.is_grad_enabled, torch.autograd.forward_ad.unpack_dual


def _no_gradient(name: str, t) -> None:
    is_grad_enabled, unpack_dual = _autograd()
    if t.requires_grad and is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which is not computed here: detach it or use torch.no_grad()")
    if unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a forward gradient, which is not computed here")


def _sizes(name: str, t) -> None:
    """The library counts in 32 bits; ctypes would drop the higher ones."""
    if t.numel() >= 2**32 and max(t.shape) >= 2**32:
        raise ValueError(f"{name} has a size of 2^32 or more: {list(t.shape)}")


def _rows(name: str, t, like, heads: int | None, tokens: int | None = None):
    """A [tokens, heads, head_dim] tensor of the dtype, device and head_dim of `like`."""
    if t.dim() != 3 or t.shape[2] != like.shape[-1]:
        raise ValueError(f"{name} must be [tokens, heads, {like.shape[-1]}], not {list(t.shape)}")
    if heads is not None and t.shape[1] != heads:
        raise ValueError(f"{name} must have {heads} heads, not {t.shape[1]}")
    if tokens is not None and t.shape[0] != tokens:
        raise ValueError(f"{name} must have {tokens} tokens, not {t.shape[0]}")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}")
    _no_gradient(name, t)
    _sizes(name, t)
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: elements of a head must be consecutive")
    return t


def _ints(name: str, t, like, shape):
    import torch
    if t.dtype != torch.int32 or t.device != like.device:
        raise ValueError(f"{name} must be int32 on {like.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    if t.numel() > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t


def _stream(device, stream) -> C.c_void_p:
    import torch
    s = stream if stream is not None else torch.cuda.current_stream(device)
    # the handle of a default stream is null on every device, so the library cannot tell
    if device.type == "cuda" and s.device != device:
        raise ValueError(f"the stream belongs to {s.device}, the tensors to {device}")
    return C.c_void_p(s.cuda_stream)


@functools.cache
def _entry(name: str):
    """An entry point without the conversions of arguments, which are C objects already."""
    from torch.autograd.graph import increment_version
    return lib()[name], increment_version


def _runner(name: str, args, keep, written):
    fn, increment_version = _entry(name)

    def run(_keep=keep):
        rc = fn(*args)
        if rc:
            check(rc)
        increment_version(written)  # a graph that saved one of them says so, as behind torch's own writes
    return run


def _span(t) -> tuple[int, int]:
    """Addresses from the first element to behind the last; (0, 0) without elements, which overlaps nothing."""
    last = 0
    for n, stride in zip(t.shape, t.stride()):
        if n == 0:
            return 0, 0
        last += (n - 1) * stride
    at = t.data_ptr()
    return at, at + (last + 1) * t.element_size()


def _overlap(a, b) -> bool:
    a, b = _span(a), _span(b)
    return a[0] < b[1] and b[0] < a[1]


def _apart(name: str, span, read) -> None:
    """What a call writes at `span` is none of what it reads, or writes otherwise: pairs of a name and a span."""
    begin, end = span
    for other, (low, high) in read:
        if begin < high and low < end:
            raise ValueError(f"{name} overlaps {other}")


def _out_rows(name: str, out, src):
    """`out` is `src` itself, or does not touch it."""
    if out.data_ptr() == src.data_ptr() and out.stride() == src.stride():
        return out
    if _overlap(out, src) and not _same_grid(out, src):
        raise ValueError(f"{name} overlaps its source: pass the source itself, or other memory")
    return out


def _same_grid(a, b) -> bool:
    """Slices of one projection (other heads of the same rows, or other ones of the parts that each head has
    there): the same strides, and never the same element."""
    if a.dim() != 3 or b.dim() != 3 or a.element_size() != b.element_size():
        return False
    low, high = sorted((a, b), key=lambda t: t.data_ptr())
    off, rest = divmod(high.data_ptr() - low.data_ptr(), a.element_size())
    if rest:
        return False
    steps = [(off, 0, 0)]  # stride, and how often each of the two takes it
    for i in range(2):
        strides = {t.stride(i) for t in (low, high) if t.shape[i] > 1}
        if len(strides) > 1:
            return False
        steps += [(n, low.shape[i], high.shape[i]) for n in strides]
    # by growing stride, each step has to reach over all that the smaller ones span
    below, above = low.shape[2], high.shape[2]
    for stride, of_low, of_high in sorted(steps, key=lambda s: (s[0], s[1] == 0)):
        if of_low == 0:  # from the one to the other: from here on both are one block
            if stride < below:
                return False
            below = above = stride + above
        else:
            if stride < max(below, above):
                return False
            below += (of_low - 1) * stride
            above += (of_high - 1) * stride
    return True


def rotary_runner(x, positions, rotary: Rotary, out=None, stream=None):
    """A prepared `rotary`."""
    out = x if out is None else out
    _rows("x", x, x, None)
    _rows("out", out, x, x.shape[1], x.shape[0])
    _out_rows("out", out, x)
    _ints("positions", positions, x, (x.shape[0],))
    _apart("out", _span(out), [("positions", _span(positions))])
    a = capi.RotaryArgs(x.data_ptr(), out.data_ptr(), x.stride(0), x.stride(1), out.stride(0), out.stride(1),
                        positions.data_ptr(), x.shape[0], x.shape[1], x.shape[2], _dtype(x))
    table = rotary.table()
    args = (C.byref(table), C.byref(a), _stream(x.device, stream))
    return _runner("mononn_rotary_apply", args, (x, out, positions, table, a), (out,))


def rotary(x, positions, rotary: Rotary, out=None, stream=None):
    """x [tokens, heads, head_dim] with the leading rotary_dim elements of each head turned by its token's
    position (int32 [tokens]); in place unless `out` is given. Returns the rotated tensor."""
    rotary_runner(x, positions, rotary, out, stream)()
    return x if out is None else out


class PagedCache:
    """Keys and values in pages.

    k_pages, v_pages  [pages, page_size, kv_heads, head_dim] f16 or bf16, with the same strides;
                      elements of a head consecutive (a head-major cache is the transposed view of
                      [pages, kv_heads, page_size, head_dim])
    page_table        int32 [sequences, most pages of a sequence]
    lengths           int32 [sequences]: tokens of each sequence, the new ones of a call among them

    What these hold may change from call to call, the tensors themselves may not: a step writes
    `cache.lengths.add_(1)` or copies into them.
    """

    def __init__(self, k_pages, v_pages, page_table, lengths):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
            raise ValueError("k_pages and v_pages must be [pages, page_size, kv_heads, head_dim], alike in sizes and strides")
        if k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device:
            raise ValueError("k_pages and v_pages must be of one dtype on one device")
        if k_pages.shape[3] > 1 and k_pages.stride(3) != 1:
            raise ValueError("k_pages: elements of a head must be consecutive")
        if page_table.dim() != 2:
            raise ValueError("page_table must be [sequences, pages]")
        _sizes("k_pages", k_pages)
        _sizes("page_table", page_table)
        n, most = page_table.shape
        _ints("page_table", page_table, k_pages, (n, most))
        _ints("lengths", lengths, k_pages, (n,))
        self._tensors = k_pages, v_pages, page_table, lengths
        self._spans = [(name, _span(t)) for name, t in zip(("k_pages", "v_pages", "page_table", "lengths"), self._tensors)]
        pages, size, heads, dim = k_pages.shape
        ps, ts, hs, _ = k_pages.stride()
        self._args = capi.PagedCacheArgs(k_pages.data_ptr(), v_pages.data_ptr(), ps, ts, hs, page_table.data_ptr(),
                                         page_table.stride(0) if n > 1 else most, lengths.data_ptr(), n, most, pages,
                                         size, heads, dim, _dtype(k_pages))

    # Read only: the addresses are taken once, so another tensor would not be seen. New contents are copied into these.
    k_pages = property(lambda self: self._tensors[0])
    v_pages = property(lambda self: self._tensors[1])
    page_table = property(lambda self: self._tensors[2])
    lengths = property(lambda self: self._tensors[3])

    @property
    def kv_heads(self) -> int:
        return self.k_pages.shape[2]

    def _pages_without_gradient(self):  # asked at each call: whether gradients are on may change behind the constructor
        _no_gradient("k_pages", self.k_pages)
        _no_gradient("v_pages", self.v_pages)

    def _indptr(self, indptr):
        return _ints("indptr", indptr, self.k_pages, (self.page_table.shape[0] + 1,))

    def append_runner(self, k, v, indptr, rotary: Rotary | None = None, positions=None, q=None, q_out=None, stream=None):
        """A prepared `append`."""
        self._pages_without_gradient()
        _rows("k", k, self.k_pages, self.kv_heads)
        _rows("v", v, self.k_pages, self.kv_heads, k.shape[0])
        self._indptr(indptr)
        if positions is not None:
            _ints("positions", positions, k, (k.shape[0],))
        if q is None and q_out is not None:
            raise ValueError("q_out without q")
        if q is not None:
            q_out = q if q_out is None else q_out
            _rows("q", q, self.k_pages, None, k.shape[0])
            _rows("q_out", q_out, self.k_pages, q.shape[1], k.shape[0])
            _out_rows("q_out", q_out, q)
            for name, t in (("k", k), ("v", v)):
                if _overlap(q_out, t) and not _same_grid(q_out, t):
                    raise ValueError(f"q_out overlaps {name}")
        given = [("indptr", _span(indptr))]
        if positions is not None:
            given.append(("positions", _span(positions)))
        if q is not None:
            at = _span(q_out)
            _apart("q_out", at, self._spans)
            _apart("q_out", at, given)
            given.append(("q", at if q_out is q else _span(q)))
        given += [("k", _span(k)), ("v", _span(v)), *self._spans[2:]]
        for name, at in self._spans[:2]:
            _apart(name, at, given)
        qs, os = (q.stride(), q_out.stride()) if q is not None else ((0, 0), (0, 0))
        a = capi.PagedAppendArgs(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                 q.data_ptr() if q is not None else None,
                                 q_out.data_ptr() if q is not None else None, qs[0], qs[1], os[0], os[1],
                                 indptr.data_ptr(), positions.data_ptr() if positions is not None else None,
                                 k.shape[0], q.shape[1] if q is not None else 0)
        table = rotary.table() if rotary is not None else None
        args = (C.byref(self._args), C.byref(table) if table is not None else None, C.byref(a),
                _stream(k.device, stream))
        return _runner("mononn_paged_append", args, (self, k, v, q, q_out, indptr, positions, table, a),
                       (self.k_pages, self.v_pages) + ((q_out,) if q is not None else ()))

    def append(self, k, v, indptr, rotary: Rotary | None = None, positions=None, q=None, q_out=None, stream=None):
        """Writes the new tokens' keys and values [tokens, kv_heads, head_dim] to their places, the last
        positions of each sequence (rows indptr[b] .. indptr[b+1]-1 are sequence b's), the keys turned by
        `rotary`; turns the queries q [tokens, q_heads, head_dim] of the same tokens in the same launch, in
        place unless `q_out` is given. `positions` (int32 [tokens]) replaces the cache's positions
        as the angle. Returns the rotated queries."""
        self.append_runner(k, v, indptr, rotary, positions, q, q_out, stream)()
        return q if q_out is None else q_out

    def attention_runner(self, q, indptr, out=None, lse=None, scale=None, causal=True, window=0, max_new=0,
                         workspace=None, stream=None):
        """A prepared `attention`; what it returns is in `out` (made here when none is given: `.out`)."""
        import torch
        self._pages_without_gradient()
        _rows("q", q, self.k_pages, None)
        self._indptr(indptr)

        def made_here(*size, dtype):  # on the stream of the call: in use there, and seen by the one of the caller
            with torch.cuda.stream(stream):
                t = torch.empty(*size, dtype=dtype, device=q.device)
            if stream is not None and t.is_cuda:
                t.record_stream(torch.cuda.current_stream(q.device))
            return t

        if out is None:
            out = made_here(q.shape, dtype=q.dtype)
        _rows("out", out, self.k_pages, q.shape[1], q.shape[0])
        if lse is not None:
            if lse.dtype != torch.float32 or lse.device != q.device or tuple(lse.shape) != tuple(q.shape[:2]) \
                    or not lse.is_contiguous():
                raise ValueError(f"lse must be contiguous float32 {list(q.shape[:2])} on {q.device}")
        if scale is not None and not C.c_float(scale).value > 0:  # 0 in 32 bits would stand for the default
            raise ValueError("scale must be positive, in 32 bits too")
        if not 0 <= window < 2**32 or not 0 <= max_new < 2**32:
            raise ValueError("window and max_new must be in 0 .. 2^32 - 1")
        if _overlap(out, q) and not _same_grid(out, q):
            raise ValueError("out overlaps q")
        taken = [*self._spans, ("indptr", _span(indptr))]
        if lse is not None:
            taken.append(("lse", _span(lse)))
            _apart("lse", taken[-1][1], [*taken[:-1], ("q", _span(q))])
        _apart("out", _span(out), taken)
        a = capi.PagedAttentionArgs(q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
                                    q.stride(0), q.stride(1), out.stride(0), out.stride(1), indptr.data_ptr(),
                                    q.shape[0], q.shape[1], 0.0 if scale is None else scale, int(causal), window,
                                    max_new, None, 0)
        need = C.c_size_t()
        check(lib().mononn_paged_attention_workspace(C.byref(self._args), C.byref(a), C.byref(need)))
        if need.value:
            if workspace is None:
                workspace = made_here(need.value, dtype=torch.uint8)
            if workspace.device != q.device or not workspace.is_contiguous():
                raise ValueError(f"workspace must be contiguous on {q.device}")
            _apart("workspace", _span(workspace), [*taken, ("q", _span(q)), ("out", _span(out))])
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        args = (C.byref(self._args), C.byref(a), _stream(q.device, stream))
        run = _runner("mononn_paged_attention", args, (self, q, out, lse, indptr, workspace, a),
                      (out,) + ((lse,) if lse is not None else ()))
        run.out = out
        return run

    def attention(self, q, indptr, out=None, lse=None, scale=None, causal=True, window=0, max_new=0, workspace=None,
                  stream=None):
        """Attention of the new tokens' queries q [tokens, q_heads, head_dim] over the cache, which holds
        their own keys already. Rows indptr[b] .. indptr[b+1]-1 are the last positions of sequence b; rows of no
        sequence stay as they were in `out` (undefined in one that is made here).
        causal: keys up to the own position; window > 0: the last `window` of those. scale: 1 / sqrt(head_dim)
        unless given. max_new: at most how many new tokens a sequence has, when known (it chooses the
        kernel). lse: float32 [tokens, q_heads] for the logarithm of the sum of exponentials. The
        workspace is allocated through torch unless given; concurrent calls need one each."""
        run = self.attention_runner(q, indptr, out, lse, scale, causal, window, max_new, workspace, stream)
        run()
        return run.out


def paged_attention_status(stream=None) -> None:
    """Waits for the stream and raises MononnError(-6) when a bounded wait expired in a paged attention
    kernel of its device since the last call (the output of that attention is incomplete)."""
    import torch
    st = stream if stream is not None else torch.cuda.current_stream()
    with torch.cuda.device(st.device):  # the handle of a default stream is null on every device
        check(lib().mononn_paged_attention_status(C.c_void_p(st.cuda_stream)))
