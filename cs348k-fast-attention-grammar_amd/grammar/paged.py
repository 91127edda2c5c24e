"""Python face of the paged key/value cache: appending new tokens
(gr_paged_append, gr_paged_append_with), attention over what is cached
(gr_paged_attn, gr_paged_attn_scaled) and reading it back (gr_paged_read).

A `PagedCache` is two tensors of pages, [pages, heads, page_size, D], a
`QuantizedPagedCache` the same with 8-bit rows and a scale for each; every call
takes either. A batch of
sequences is described by three int32 tensors on the GPU: `table` [B, width],
each sequence's page ids in order; `lens` [B], its keys, the new tokens' among
them; and for packed batches `starts` [B + 1], the first row of each sequence's
new tokens. New token i of n stands at position len - n + i. Uniform batches
are [B, heads, n, D] like the framework's other attention calls, packed ones
[rows, heads, D]; rows of a packed batch that belong to no sequence are neither
read nor written. A decode step is paged_append and paged_attention with n = 1,
a prompt the same two calls with its tokens, whole or in chunks, and both may
share a packed batch. The reference has no cache (its attention takes as many
keys as queries, run_attention_search.py:34-114).

Lengths, starts and page ids are read on the GPU, so one bound or captured call
serves every step. What lies outside of the cache or the table is not touched:
such keys do not exist. The results carry no gradient. There is no CPU path: CPU
tensors or a missing library raise.
"""
from __future__ import annotations

import ctypes
import functools
import math

from . import runtime as rt
from .norm import HeadNorm
from .rotary import Rotary, _head_strides, _takes, check_out, check_positions, head_strides


class PagedCache:
    """Key and value pages: tensors [pages, heads, page_size, D] of one shape,
    fp16 or bf16, D 64 or 128, page_size a power of two from 16 on, unit stride
    along D, other strides multiples of 8 (so [pages, page_size, heads, D]
    storage serves, transposed)."""

    def __init__(self, k, v):
        for name, t in (("k", k), ("v", v)):
            if not t.is_cuda:
                raise ValueError(f"PagedCache: {name} must be a GPU tensor (no CPU path)")
            if t.dim() != 4 or t.shape != k.shape or t.dtype != k.dtype or t.device != k.device or t.stride(3) != 1:
                raise ValueError("PagedCache: k and v must be [pages, heads, page_size, D] of one shape, dtype and "
                                 "device with unit stride on D")
            if t.shape[0] and any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
                raise ValueError("PagedCache: pages of k and v must not overlap (a stride of 0)")
        pages, heads, size, D = k.shape
        if rt.dtype_code(k.dtype) == rt.GR_F32:
            raise ValueError("PagedCache: fp16 or bf16")
        if max(pages, heads) >= 1 << 31:
            raise ValueError(f"PagedCache: {pages} pages of {heads} heads are too many (2^31)")
        if D not in (64, 128) or size < 16 or size & (size - 1) or size > 1 << 20:
            raise ValueError(f"PagedCache: D {D} must be 64 or 128 and page_size {size} a power of two from 16 to 2^20")
        self.k, self.v, self.dtype, self.index = k, v, k.dtype, k.get_device()
        self.pages, self.heads, self.page_size, self.head_dim = pages, heads, size, D
        self.scales_ref = None
        self.desc = rt.PagedCacheDesc(k.data_ptr(), v.data_ptr(), rt._ll3(*k.stride()[:3]), rt._ll3(*v.stride()[:3]),
                                      rt.dtype_code(k.dtype), pages, heads, size, D)
        self.ref = ctypes.addressof(self.desc)

    def __reduce__(self):
        """For copies and pickles: the descriptor points at this object's pages."""
        return type(self), (self.k, self.v)

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, head_dim: int, dtype, device="cuda"):
        """A cache of unwritten pages (their contents are never read before
        they are appended to)."""
        import torch
        shape = (pages, heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


class QuantizedPagedCache:
    """Key and value pages of 8-bit rows: k and v torch.float8_e4m3fn [pages, heads,
    page_size, D], as PagedCache's but with strides that are multiples of 16;
    scales torch.float8_e8m0fnu [pages, heads, 2, page_size], a power of two for each
    key's (index 0) and value's (1) row, unit stride along the slots, other strides
    multiples of 16. dtype: fp16 or
    bf16, the tokens'.

    A row x is held as round(x / scale), scale the least power of two (2^-127 at
    least) by which its largest magnitude is at most 448: four significant
    bits, off by at most 2^-4 of each element or, where that is more, 2^-10 of the scale (of
    an element below 2^-6 of it; 2^-17.8 of the row's largest magnitude, if that is 2^-119
    or more). Rows are clamped to 61440 (fp16) or 15 2^124 (bf16) first, so that none
    stands for more than the tokens' type holds. A row with a value that is not finite becomes NaN.

    Attention and paged_read take a row's numbers times its scale in the tokens' type. Where
    that has no such number, the nearest one is taken, a whole number of 2^-24 (fp16) or 2^-133
    (bf16): under scales below 2^-15 or 2^-124, which tokens of the type stored as they are do
    not need, but keys that a norm or a rotation made small have (in fp16, rows of at most 448
    2^-16)."""

    def __init__(self, k, v, scales, dtype):
        import torch
        for name, t, want in (("k", k, torch.float8_e4m3fn), ("v", v, torch.float8_e4m3fn),
                              ("scales", scales, torch.float8_e8m0fnu)):
            if not t.is_cuda:
                raise ValueError(f"QuantizedPagedCache: {name} must be a GPU tensor (no CPU path)")
            if t.dim() != 4 or t.dtype != want or t.device != k.device or (t.stride(3) != 1 and t.shape[3] > 1):
                raise ValueError(f"QuantizedPagedCache: {name} must be a 4-D {want} tensor on {k.device} with unit stride")
            if 0 not in t.shape and any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
                raise ValueError("QuantizedPagedCache: pages of k, v and scales must not overlap (a stride of 0)")
        pages, heads, size, D = k.shape
        if v.shape != k.shape or scales.shape != (pages, heads, 2, size):
            raise ValueError(f"QuantizedPagedCache: k, v and scales must be [pages, heads, page_size, D] twice and [pages, heads, 2, "
                             f"page_size], not {tuple(k.shape)}, {tuple(v.shape)} and {tuple(scales.shape)}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("QuantizedPagedCache: tokens of fp16 or bf16")
        if max(pages, heads) >= 1 << 31:
            raise ValueError(f"QuantizedPagedCache: {pages} pages of {heads} heads are too many (2^31)")
        if D not in (64, 128) or size < 16 or size & (size - 1) or size > 1 << 20:
            raise ValueError(f"QuantizedPagedCache: D {D} must be 64 or 128 and page_size {size} a power of two from 16 to 2^20")
        self.k, self.v, self.scales, self.dtype, self.index = k, v, scales, dtype, k.get_device()
        self.pages, self.heads, self.page_size, self.head_dim = pages, heads, size, D
        self.desc = rt.PagedCacheDesc(k.data_ptr(), v.data_ptr(), rt._ll3(*k.stride()[:3]), rt._ll3(*v.stride()[:3]),
                                      rt.dtype_code(dtype), pages, heads, size, D)
        self.scales_desc = rt.PagedScales(scales.data_ptr(), rt._ll3(*scales.stride()[:3]))
        self.ref, self.scales_ref = ctypes.addressof(self.desc), ctypes.addressof(self.scales_desc)

    def __reduce__(self):
        """For copies and pickles: the descriptors point at this object's pages. (As
        bytes: torch does not pickle 8-bit floating-point tensors.)"""
        import torch
        return type(self)._of_bytes, (*(t.view(torch.uint8) for t in (self.k, self.v, self.scales)), self.dtype)

    @classmethod
    def _of_bytes(cls, k, v, scales, dtype):
        import torch
        return cls(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), dtype)

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, head_dim: int, dtype, device="cuda"):
        """A cache of unwritten pages for tokens of `dtype`."""
        import torch
        k, v = (torch.empty((pages, heads, page_size, head_dim), dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        return cls(k, v, torch.empty((pages, heads, 2, page_size), dtype=torch.float8_e8m0fnu, device=device), dtype)


@functools.lru_cache(maxsize=4096)
def _batch_sizes(table: tuple, table_st: tuple, lens: tuple, lens_st: tuple, starts, starts_st, x: tuple):
    """(B, width, leading sizes of the tokens) of a call's shapes and strides, or what is wrong with them."""
    for n, shape, st, dim in (("table", table, table_st, 2), ("lens", lens, lens_st, 1), ("starts", starts, starts_st, 1)):
        if shape is not None and (len(shape) != dim or (st[-1] != 1 and shape[-1] > 1)):
            return f"{n} must be a {dim}-D int32 tensor with unit stride"
    B, width = table
    if max(B, width, *x) >= 1 << 31:                                                # (C integers would wrap)
        return f"{tuple(x)} by a table {tuple(table)} is too large for one call (2^31)"
    if lens[0] != B or B == 0 or width == 0:
        return f"table {tuple(table)} and lens {tuple(lens)} do not describe a batch"
    if starts is None:
        return (B, width, (B, x[2])) if len(x) == 4 and x[0] == B else \
            f"the tokens must be [{B}, heads, n, D] (packed rows need starts), not {tuple(x)}"
    return (B, width, (x[0],)) if len(x) == 3 and starts[0] == B + 1 else \
        f"with starts [{B + 1}] the tokens must be packed [rows, heads, D], not {tuple(x)}"


def _batch(cache, table, lens, starts, x, max_new, max_len, who):
    """(gr_paged_batch, leading sizes of the tokens) of a call on `x`: [B, heads,
    n, D] or, with starts, [rows, heads, D]."""
    import torch
    index, int32 = cache.index, torch.int32
    if starts is None:
        sizes = _batch_sizes(table.shape, table.stride(), lens.shape, lens.stride(), None, None, x.shape)
        at, ok = None, True
    else:
        sizes = _batch_sizes(table.shape, table.stride(), lens.shape, lens.stride(), starts.shape, starts.stride(), x.shape)
        at, ok = starts.data_ptr(), starts.dtype == int32 and starts.get_device() == index
    if not ok or table.dtype != int32 or lens.dtype != int32 or table.get_device() != index or lens.get_device() != index:
        raise ValueError(f"{who}: table, lens and starts must be int32 tensors on {cache.k.device}")
    if type(sizes) is str:
        raise ValueError(f"{who}: {sizes}")
    B, width, lead = sizes
    return rt.PagedBatch(table.data_ptr(), table.stride(0), lens.data_ptr(), at, B, lead[-1], width, int(max_new),
                         int(max_len)), lead


@functools.lru_cache(maxsize=4096)
def _heads_strides(shape: tuple, st: tuple, lead: tuple, heads: int, dim: int):
    """{batch, token, head} strides of `heads` heads of the tokens `lead`; None: another shape."""
    if shape != ((lead[0], heads, lead[1], dim) if len(lead) == 2 else (lead[0], heads, dim)):
        return None
    return _head_strides(shape, st) or "stride"


def _heads(t, name, lead, heads, cache, who):
    """The strides of `heads` heads of the tokens `lead`, checked."""
    st = _heads_strides(t.shape, t.stride(), lead, heads, cache.head_dim)
    if st is None or t.dtype != cache.dtype or t.get_device() != cache.index:
        want = (*lead[:1], heads, *lead[1:], cache.head_dim)
        raise ValueError(f"{who}: {name} must be {want} {cache.dtype} on {cache.k.device} (no CPU path), not "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return st if st != "stride" else head_strides(t, name, who)


def _append_args(k, v, cache, table, lens, starts, q, rotary, norm, positions, max_new, out, stream):
    """(function, its arguments, the queries' result, what the arguments point to)"""
    who = "paged_append"
    desc, lead = _batch(cache, table, lens, starts, k, max_new, 0, who)
    ks, vs = _heads(k, "k", lead, cache.heads, cache, who), _heads(v, "v", lead, cache.heads, cache, who)
    if rotary is None:
        if (q is not None and norm is None) or positions is not None:
            raise ValueError(f"{who}: q is only rotated or normed here, and positions only turn: they need `rotary` or `norm`")
        ref = None
    elif rotary.head_dim != cache.head_dim or rotary.index != cache.index:
        raise ValueError(f"{who}: the rotation is for heads of {rotary.head_dim} on {rotary.device}")
    else:
        ref = rotary.ref
    if q is not None:
        Hq = q.shape[1] if q.dim() >= 3 else 0
        qs, out = _heads(q, "q", lead, Hq, cache, who), check_out(out, q, "out", who, stream)
        qp, op, os = q.data_ptr(), out.data_ptr(), head_strides(out, "out", who)
    elif out is None:
        qp = op = qs = os = None
        Hq = 0
    else:
        raise ValueError(f"{who}: `out` is the queries' and needs q")
    pp, ps = (None, None) if positions is None else (positions.data_ptr(), check_positions(positions, rotary, lead, who))
    args = (qp, op, Hq, qs, os, k.data_ptr(), v.data_ptr(), ks, vs, pp, ps)
    keep = (desc, k, v, cache, table, lens, starts, q, rotary, positions, out)
    if norm is None and cache.scales_ref is None:
        return rt.lib().gr_paged_append, (cache.ref, ctypes.addressof(desc), ref) + args, out, keep
    spec = None if norm is None else norm.spec(cache.head_dim, cache.dtype, cache.index, who)
    args = (cache.ref, cache.scales_ref, ctypes.addressof(desc), ref, None if spec is None else ctypes.addressof(spec)) + args
    return rt.lib().gr_paged_append_with, args, out, keep + (spec,) + (() if norm is None else (norm.q_weight, norm.k_weight))


def paged_append(k, v, cache: PagedCache | QuantizedPagedCache, table, lens, *, starts=None, q=None,
                 rotary: Rotary | None = None, norm: HeadNorm | None = None, positions=None, max_new: int = 0, out=None,
                 stream=None):
    """Puts the new tokens' keys and values into their pages, in one launch: as they
    are, or quantised (QuantizedPagedCache) after norm and rotation, from fp32.

    k, v: [B, heads, n, D], or [rows, heads, D] with `starts`; any strides that
    are multiples of 8, unit on D (slices of a projection's output serve).
    rotary: a `Rotary` that turns the keys on the way, and q ([.., Hq, .., D]) if
    given, into a new tensor laid out as q or into `out` (which may be q and
    shares no other memory with the call's tensors; nor do k and v lie in pages
    that the call writes).
    norm: a `HeadNorm` that norms the keys, and q if given, before they are turned.
    positions: int32, [B, n], [n] or (packed) [rows], with several axes led by
    them; default: each token's place len - n + i, on every axis.
    Returns the rotated queries, or None without q. A token whose place is
    outside of the table or on a page id outside of the cache is not stored.
    max_new: as paged_attention takes it, so that one set of arguments serves
    both; an append is shared out alike whatever it is."""
    fn, args, out, keep = _append_args(k, v, cache, table, lens, starts, q, rotary, norm, positions, max_new, out, stream)
    rt.launch(fn, args, k, stream, "gr_paged_append")
    return out


def bind_paged_append(k, v, cache: PagedCache | QuantizedPagedCache, table, lens, *, starts=None, q=None,
                      rotary: Rotary | None = None, norm: HeadNorm | None = None, positions=None, max_new: int = 0,
                      out=None, stream=None):
    """Validate once and return (launch, out): launch() enqueues the append
    on these tensors with pre-packed arguments; arguments as paged_append."""
    fn, args, out, keep = _append_args(k, v, cache, table, lens, starts, q, rotary, norm, positions, max_new, out, stream)
    return rt.launcher(fn, args, k, stream, "gr_paged_append", out, keep), out


def _attn_args(q, cache, table, lens, starts, causal, scale, max_new, max_len, out, lse, workspace, stream):
    import torch
    who = "paged_attention"
    desc, lead = _batch(cache, table, lens, starts, q, max_new, max_len, who)
    Hq = q.shape[1]
    qs = _heads(q, "q", lead, Hq, cache, who)
    if Hq == 0 or Hq % cache.heads:
        raise ValueError(f"{who}: {Hq} query heads are not a multiple of the cache's {cache.heads}")
    out = check_out(out, q, "out", who, stream)
    if lse is not None:
        want = (lead[0], lead[1], Hq) if len(lead) == 2 else (lead[0], Hq)
        if tuple(lse.shape) != want or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.get_device() != cache.index:
            raise ValueError(f"{who}: lse must be a contiguous {want} float32 tensor")
    if scale is None:
        scale = 1.0 / math.sqrt(cache.head_dim)
    ref, scales = ctypes.addressof(desc), cache.scales_ref
    if scales is None:
        fn, head, need = rt.lib().gr_paged_attn, (cache.ref,), int(rt.lib().gr_paged_attn_workspace(cache.ref, ref, Hq))
    else:
        fn, head = rt.lib().gr_paged_attn_scaled, (cache.ref, scales)
        need = int(rt.lib().gr_paged_attn_scaled_workspace(cache.ref, scales, ref, Hq))
    if workspace is not None and (workspace.get_device() != cache.index or not workspace.is_contiguous()):
        raise ValueError(f"{who}: workspace must be a contiguous tensor on {cache.k.device}")
    if need and workspace is None:
        workspace = rt.workspace(need, q.device, stream)
    size = workspace.numel() * workspace.element_size() if workspace is not None else 0
    args = head + (ref, q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None, Hq,
            qs, head_strides(out, "out", who), int(bool(causal)), float(scale),
            workspace.data_ptr() if workspace is not None else None, size)
    return fn, args, out, (desc, q, cache, table, lens, starts, out, lse, workspace)


def paged_attention(q, cache: PagedCache | QuantizedPagedCache, table, lens, *, starts=None, causal: bool = True,
                    scale: float | None = None, max_new: int = 0, max_len: int = 0, out=None, lse=None, workspace=None,
                    stream=None):
    """O = softmax(scale * Q K^T) V of the new tokens over the cached keys.

    q: [B, Hq, n, D], or [rows, Hq, D] with `starts`; Hq a multiple of the
    cache's heads, query head h reading key head h // (Hq / heads). Token i
    of n sees the keys up to its own place len - n + i (causal=True) or all len
    keys. A row that sees none gets 0.
    max_new, max_len: the most new tokens and keys of a sequence, where known;
    they only choose how the work is shared out.
    lse: float32 [B, n, Hq] or [rows, Hq] to receive the log-sum-exp of the scaled
    scores (natural log). workspace: device memory for calls whose keys are
    shared out (allocated here unless given; rt.lib().gr_paged_attn_workspace, for a
    quantised cache gr_paged_attn_scaled_workspace, names the size; with less the keys are shared out less).
    Returns the result, laid out as q, or `out`, which may be q and shares no
    other memory with the call's tensors."""
    fn, args, out, keep = _attn_args(q, cache, table, lens, starts, causal, scale, max_new, max_len, out, lse, workspace,
                                     stream)
    rt.launch(fn, args, q, stream, "gr_paged_attn")
    return out


def bind_paged_attention(q, cache: PagedCache | QuantizedPagedCache, table, lens, *, starts=None, causal: bool = True,
                         scale: float | None = None, max_new: int = 0, max_len: int = 0, out=None, lse=None,
                         workspace=None, stream=None):
    """Validate once and return (launch, out): launch() enqueues the attention on
    these tensors with pre-packed arguments and the workspace allocated here, for
    loops on fixed buffers; arguments as paged_attention. Launches of one binding
    share its workspace: those that may overlap in time (two streams, two
    captured graphs) need bindings of their own."""
    fn, args, out, keep = _attn_args(q, cache, table, lens, starts, causal, scale, max_new, max_len, out, lse, workspace,
                                     stream)
    return rt.launcher(fn, args, q, stream, "gr_paged_attn", out, keep), out


def paged_read(cache: PagedCache | QuantizedPagedCache, table, lens, length: int | None = None, *, starts=None,
               k_out=None, v_out=None, stream=None):
    """The sequences' keys and values as dense tensors of the cache's dtype, in one
    launch.

    table, lens: as paged_attention takes them. Without `starts` the result is (k, v)
    [B, heads, length, D], key j of a sequence at place j and zeros behind its
    end; with starts, int32 [B + 1] on the GPU, it is packed, [rows, heads, D], key j of
    sequence b in row starts[b] + j, zeros behind its end up to starts[b + 1]; rows of no
    sequence are left alone.
    k_out, v_out: where the results go (both or neither; packed calls need them, and their size says
    length or rows). They share no memory with each other or the cache. Keys on a
    page id outside of the cache, or outside of the table, read as zeros."""
    who = "paged_read"
    if (k_out is None) != (v_out is None):
        raise ValueError(f"{who}: k_out and v_out come together")
    made = k_out is None
    if made:
        if starts is not None or length is None or int(length) < 0:
            raise ValueError(f"{who}: needs a length, or k_out and v_out")
        shape = (table.shape[0] if table.dim() == 2 else 0, cache.heads, int(length), cache.head_dim)
        k_out, v_out = rt.result(shape, cache.dtype, cache.k.device, stream), rt.result(shape, cache.dtype, cache.k.device, stream)
    elif length is not None and (starts is not None or k_out.dim() != 4 or k_out.shape[2] != length):
        raise ValueError(f"{who}: k_out {tuple(k_out.shape)} is not of length {length}")
    desc, lead = _batch(cache, table, lens, starts, k_out, 0, 0, who)
    ks = vs = _heads(k_out, "k_out", lead, cache.heads, cache, who)
    if not made:
        vs = _heads(v_out, "v_out", lead, cache.heads, cache, who)
        for t in (k_out, v_out):
            if not _takes(t.shape, t.stride(), t.shape):
                raise ValueError(f"{who}: k_out and v_out must not overlap themselves (a stride of 0)")
    if k_out.numel() == 0:
        return k_out, v_out
    rt.launch(rt.lib().gr_paged_read, (cache.ref, cache.scales_ref, ctypes.addressof(desc), k_out.data_ptr(),
                                       v_out.data_ptr(), ks, vs), k_out, stream, "gr_paged_read")
    return k_out, v_out
