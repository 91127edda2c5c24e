"""Python face of the paged key/value cache: appending new tokens
(gr_paged_append) and attention over what is cached (gr_paged_attn).

A `PagedCache` is two tensors of pages, [pages, heads, page_size, D]. A batch of
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
from .rotary import Rotary, _head_strides, check_out, check_positions, head_strides


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


def _append_args(k, v, cache, table, lens, starts, q, rotary, positions, max_new, out, stream):
    who = "paged_append"
    desc, lead = _batch(cache, table, lens, starts, k, max_new, 0, who)
    ks, vs = _heads(k, "k", lead, cache.heads, cache, who), _heads(v, "v", lead, cache.heads, cache, who)
    if rotary is None:
        if q is not None or positions is not None:
            raise ValueError(f"{who}: q is only rotated here, and positions only turn: both need `rotary`")
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
    args = (cache.ref, ctypes.addressof(desc), ref, qp, op, Hq, qs, os, k.data_ptr(), v.data_ptr(), ks, vs, pp, ps)
    return args, out, (desc, k, v, cache, table, lens, starts, q, rotary, positions, out)


def paged_append(k, v, cache: PagedCache, table, lens, *, starts=None, q=None, rotary: Rotary | None = None,
                 positions=None, max_new: int = 0, out=None, stream=None):
    """Puts the new tokens' keys and values into their pages, in one launch.

    k, v: [B, heads, n, D], or [rows, heads, D] with `starts`; any strides that
    are multiples of 8, unit on D (slices of a projection's output serve).
    rotary: a `Rotary` that turns the keys on the way, and q ([.., Hq, .., D]) if
    given, into a new tensor laid out as q or into `out` (which may be q and
    shares no other memory with the call's tensors; nor do k and v lie in pages
    that the call writes).
    positions: int32, [B, n], [n] or (packed) [rows], with several axes led by
    them; default: each token's place len - n + i, on every axis.
    Returns the rotated queries, or None without q. A token whose place is
    outside of the table or on a page id outside of the cache is not stored.
    max_new: as paged_attention takes it, so that one set of arguments serves
    both; an append is shared out alike whatever it is."""
    args, out, keep = _append_args(k, v, cache, table, lens, starts, q, rotary, positions, max_new, out, stream)
    rt.launch(rt.lib().gr_paged_append, args, k, stream, "gr_paged_append")
    return out


def bind_paged_append(k, v, cache: PagedCache, table, lens, *, starts=None, q=None, rotary: Rotary | None = None,
                      positions=None, max_new: int = 0, out=None, stream=None):
    """Validate once and return (launch, out): launch() enqueues gr_paged_append
    on these tensors with pre-packed arguments; arguments as paged_append."""
    args, out, keep = _append_args(k, v, cache, table, lens, starts, q, rotary, positions, max_new, out, stream)
    return rt.launcher(rt.lib().gr_paged_append, args, k, stream, "gr_paged_append", out, keep), out


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
    ref = ctypes.addressof(desc)
    need = int(rt.lib().gr_paged_attn_workspace(cache.ref, ref, Hq))
    if workspace is not None and (workspace.get_device() != cache.index or not workspace.is_contiguous()):
        raise ValueError(f"{who}: workspace must be a contiguous tensor on {cache.k.device}")
    if need and workspace is None:
        workspace = rt.workspace(need, q.device, stream)
    size = workspace.numel() * workspace.element_size() if workspace is not None else 0
    args = (cache.ref, ref, q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None, Hq,
            qs, head_strides(out, "out", who), int(bool(causal)), float(scale),
            workspace.data_ptr() if workspace is not None else None, size)
    return args, out, (desc, q, cache, table, lens, starts, out, lse, workspace)


def paged_attention(q, cache: PagedCache, table, lens, *, starts=None, causal: bool = True, scale: float | None = None,
                    max_new: int = 0, max_len: int = 0, out=None, lse=None, workspace=None, stream=None):
    """O = softmax(scale * Q K^T) V of the new tokens over the cached keys.

    q: [B, Hq, n, D], or [rows, Hq, D] with `starts`; Hq a multiple of the
    cache's heads, query head h reading key head h // (Hq / heads). Token i
    of n sees the keys up to its own place len - n + i (causal=True) or all len
    keys. A row that sees none gets 0.
    max_new, max_len: the most new tokens and keys of a sequence, where known;
    they only choose how the work is shared out.
    lse: float32 [B, n, Hq] or [rows, Hq] to receive the log-sum-exp of the scaled
    scores (natural log). workspace: device memory for calls whose keys are
    shared out (allocated here unless given; rt.lib().gr_paged_attn_workspace
    names the size; with less the keys are shared out less).
    Returns the result, laid out as q, or `out`, which may be q and shares no
    other memory with the call's tensors."""
    args, out, keep = _attn_args(q, cache, table, lens, starts, causal, scale, max_new, max_len, out, lse, workspace,
                                 stream)
    rt.launch(rt.lib().gr_paged_attn, args, q, stream, "gr_paged_attn")
    return out


def bind_paged_attention(q, cache: PagedCache, table, lens, *, starts=None, causal: bool = True,
                         scale: float | None = None, max_new: int = 0, max_len: int = 0, out=None, lse=None,
                         workspace=None, stream=None):
    """Validate once and return (launch, out): launch() enqueues gr_paged_attn on
    these tensors with pre-packed arguments and the workspace allocated here, for
    loops on fixed buffers; arguments as paged_attention. Launches of one binding
    share its workspace: those that may overlap in time (two streams, two
    captured graphs) need bindings of their own."""
    args, out, keep = _attn_args(q, cache, table, lens, starts, causal, scale, max_new, max_len, out, lse, workspace,
                                 stream)
    return rt.launcher(rt.lib().gr_paged_attn, args, q, stream, "gr_paged_attn", out, keep), out
