"""Python face of the position rotation of queries and keys (gr_rotary).

`rotary(q, k, positions, rot)` turns the pairs of every head by position times
frequency, differentiably; `rotary_fwd` is the launch alone, for callers that
give the output tensors. `Rotary` holds what a model fixes once: which elements
of a head form pairs, their frequencies and, for images and video, which
position axis (time, height, width) each pair turns with. The reference has no
positions; its attention (run_attention_search.py:34-114) is what the rotated
heads go to.

There is no CPU path: CPU tensors or a missing library raise.
"""
from __future__ import annotations

import ctypes
import functools
import math

from . import runtime as rt

_pair = functools.lru_cache(maxsize=1024)(lambda *s: (ctypes.c_longlong * len(s))(*s))


_PI_BITS = 1216


@functools.lru_cache(maxsize=None)
def _pi() -> int:
    """pi 2^1216, by Machin's formula pi / 4 = 4 arctan(1/5) - arctan(1/239) in
    integers with 32 bits more (a few hundred terms, each off by less than 2)."""
    def arctan(x):
        term = (1 << (_PI_BITS + 32)) // x
        total, n, sign = term, 1, 1
        while term:
            term //= x * x
            n, sign = n + 2, -sign
            total += sign * (term // n)
        return total
    return 4 * (4 * arctan(5) - arctan(239)) >> 32


def _turns(f: float) -> int:
    """f radians as a whole number of 2^-64 turns, modulo one turn: the nearest
    to the double's own value, whatever its size (a quotient in doubles would be
    off by 2^-56 of a turn at 1 radian, which position 2^31 makes 2^-25)."""
    n, d = f.as_integer_ratio()
    num, den = n << (63 + _PI_BITS), d * _pi()                # f 2^64 / (2 pi)
    return (2 * num + den) // (2 * den) % (1 << 64)


class Rotary:
    """The rotation of heads of `head_dim` elements.

    rotary_dim: the first elements of a head that are rotated (a multiple of
    16; default: all). Pair j is elements j and j + rotary_dim / 2, or 2j and
    2j + 1 with interleaved=True.
    sections: how many pairs turn with each position axis, in order (default:
    all with one axis; at most 8 axes).
    Frequencies, radians a position: base ** (-j / pairs) for pair j of all
    pairs, or with per_axis=True base ** (-j / n) for pair j of the n of an axis;
    inv_freq (one number a pair) replaces them.
    device: where the tables of this object live (one object a GPU)."""

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, base: float = 10000.0, sections=None,
                 per_axis: bool = False, interleaved: bool = False, inv_freq=None, device="cuda"):
        import torch
        rd = head_dim if rotary_dim is None else int(rotary_dim)
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"Rotary: head_dim {head_dim} must be a multiple of 16 up to 256")
        if rd % 16 or not 16 <= rd <= head_dim:
            raise ValueError(f"Rotary: rotary_dim {rd} must be a multiple of 16 up to head_dim {head_dim}")
        pairs = rd // 2
        sections = [pairs] if sections is None else [int(s) for s in sections]
        if not 1 <= len(sections) <= 8 or min(sections) < 0 or sum(sections) != pairs:
            raise ValueError(f"Rotary: sections {sections} must be 1 to 8 counts that sum to the {pairs} pairs")
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
        if inv_freq is None:
            if not base > 0:
                raise ValueError(f"Rotary: base {base} must be positive")
            place = [j / n for n in sections for j in range(n)] if per_axis else [j / pairs for j in range(pairs)]
            freqs = [float(base) ** -x for x in place]
        else:
            freqs = [float(f) for f in (inv_freq.tolist() if hasattr(inv_freq, "tolist") else inv_freq)]
            if len(freqs) != pairs or not all(math.isfinite(f) for f in freqs):
                raise ValueError(f"Rotary: inv_freq must be {pairs} finite numbers")
        self.head_dim, self.rotary_dim, self.interleaved = int(head_dim), rd, bool(interleaved)
        self.sections, self.naxes = tuple(sections), len(sections)
        self.inv_freq = tuple(freqs)
        # turns a position, modulo one, as whole numbers of 2^-64 (two's complement)
        whole = [_turns(f) for f in freqs]
        self.turns = torch.tensor([w - (1 << 64) if w >> 63 else w for w in whole], dtype=torch.int64, device=device)
        self.axes = torch.tensor(axes, dtype=torch.uint8, device=device)
        self._describe()

    def _describe(self):
        self.device, self.index = self.turns.device, self.turns.get_device()
        self.desc = rt.RotarySpec(self.turns.data_ptr(), self.axes.data_ptr(), self.rotary_dim // 2, self.naxes,
                                  self.head_dim, int(self.interleaved))
        self.ref = ctypes.addressof(self.desc)

    def __getstate__(self):
        """For copies and pickles: without what points at this object's tables."""
        return {n: v for n, v in self.__dict__.items() if n not in ("device", "index", "desc", "ref")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._describe()


@functools.lru_cache(maxsize=1024)
def _position_strides(naxes: int, shape: tuple, st: tuple, lead: tuple):
    """{axis, batch, token} strides of positions of `shape`, None if it does not fit the tokens `lead`."""
    axis = 0
    if naxes > 1:
        if shape[:1] != (naxes,):
            return None
        axis, shape, st = st[0], shape[1:], st[1:]
    if shape == lead:
        return _pair(axis, *((0,) * (2 - len(st))), *st)
    return _pair(axis, 0, st[0]) if len(lead) == 2 and shape == lead[1:] else None


def check_positions(positions, rot, lead: tuple, who: str):
    """The strides {axis, batch, token} of int32 `positions`: [*lead] or, with
    several axes, [axes, *lead]; a batch of positions may be left out."""
    import torch
    if positions.dtype != torch.int32 or positions.get_device() != rot.index:
        raise ValueError(f"{who}: positions must be an int32 tensor on {rot.device}")
    ps = _position_strides(rot.naxes, positions.shape, positions.stride(), lead)
    if ps is None:
        raise ValueError(f"{who}: positions {tuple(positions.shape)} do not match the tokens {lead}"
                         + (f" led by the {rot.naxes} axes" if rot.naxes > 1 else ""))
    return ps


@functools.lru_cache(maxsize=4096)
def _head_strides(shape: tuple, st: tuple):
    if st[-1] != 1:
        return None
    st = [s if n > 1 else 0 for s, n in zip(st, shape)]                # a single row's stride says nothing
    return _pair(st[0], st[2], st[1]) if len(st) == 4 else _pair(0, st[0], st[1])


def head_strides(t, name: str, who: str):
    """{batch, token, head} strides of [B, H, N, D] or packed [T, H, D] heads."""
    st = _head_strides(t.shape, t.stride())
    if st is None:
        raise ValueError(f"{who}: {name} must have unit stride on its last dimension")
    return st


@functools.lru_cache(maxsize=4096)
def _takes(shape: tuple, st: tuple, like: tuple) -> bool:
    return shape == like and not any(s == 0 and n > 1 for s, n in zip(st, shape))


def check_out(out, like, name: str, who: str, stream):
    """`out`, checked, or a new tensor laid out as `like` for a launch on `stream`."""
    import torch
    if out is None:
        return rt.empty_like(like, stream) if stream is not None else torch.empty_like(like)
    if not _takes(out.shape, out.stride(), like.shape) or out.dtype != like.dtype or out.get_device() != like.get_device():
        raise ValueError(f"{who}: bad `{name}` tensor")
    return out


@functools.lru_cache(maxsize=4096)
def _tokens(q: tuple, q_st: tuple, k, k_st, dim: int):
    """(B, N, query heads, their strides, key heads, theirs) of a call's shapes and strides, None if they do not fit."""
    for shape, st in ((q, q_st), (k, k_st)):
        if shape is not None and (len(shape) != 4 or shape[3] != dim or st[3] != 1 or shape[0] != q[0] or shape[2] != q[2]):
            return None
        if shape is not None and max(shape[0] * shape[2], shape[1]) >= 1 << 31:     # (C integers would wrap)
            return "too many"
    return (q[0], q[2], q[1], _head_strides(q, q_st)) + ((0, None) if k is None else (k[1], _head_strides(k, k_st)))


def rotary_fwd(q, k, positions, rot: Rotary, *, inverse: bool = False, out=None, k_out=None, stream=None):
    """q [B, Hq, N, D] and k [B, Hk, N, D] (or None) rotated to `positions`: int32,
    [N] or [B, N], with several axes [axes, N] or [axes, B, N]. fp16, bf16 or
    fp32 on the GPU, any strides that are multiples of 8 with a unit one on D.
    Returns (q', k'), new tensors laid out as the given ones, or `out` and
    `k_out`, which may be q and k themselves and share no other memory with them
    or each other. inverse=True rotates back."""
    who = "rotary"
    if q is None:
        raise ValueError(f"{who}: q must be given")
    index = rot.index
    ok = index >= 0 and q.get_device() == index
    if k is None:
        sizes = _tokens(q.shape, q.stride(), None, None, rot.head_dim)
    else:
        sizes = _tokens(q.shape, q.stride(), k.shape, k.stride(), rot.head_dim)
        ok = ok and k.get_device() == index and k.dtype == q.dtype
    if sizes is None or not ok:
        raise ValueError(f"{who}: q and k must be [B, H, N, {rot.head_dim}] tensors of one dtype, B and N on {rot.device} "
                         "(no CPU path) with unit stride on their last dimension")
    if sizes == "too many":
        raise ValueError(f"{who}: {tuple(q.shape)} is too many tokens or heads for one call (2^31)")
    B, N, Hq, qs, Hk, ks = sizes
    ps = check_positions(positions, rot, (B, N), who)
    out = check_out(out, q, "out", who, stream)
    head = (rot.ref, q.data_ptr(), out.data_ptr(), Hq, qs, head_strides(out, "out", who))
    if k is None:
        head += (None, None, 0, None, None)
    else:
        k_out = check_out(k_out, k, "k_out", who, stream)
        k_to = k_out.data_ptr()
        if k_to == head[2] and k_to:
            raise ValueError(f"{who}: `out` and `k_out` must be two tensors")
        head += (k.data_ptr(), k_to, Hk, ks, head_strides(k_out, "k_out", who))
    if B == 0 or N == 0:
        return out, k_out
    rt.launch(rt.lib().gr_rotary, head + (rt.dtype_code(q.dtype), B, N, positions.data_ptr(), ps, int(bool(inverse))),
              q, stream, "gr_rotary")
    return out, k_out


@functools.lru_cache(maxsize=1024)
def _is_dense(shape: tuple, st: tuple) -> bool:
    return st[3] == 1 and all(n == 1 or (s > 0 and s % 8 == 0) for s, n in zip(st, shape[:3]))


def _dense(t):
    """t with strides the kernels take: itself, or a contiguous copy (the
    gradient of a sum is a broadcast one, of a slice a strided one)."""
    if t.dim() != 4 or (_is_dense(t.shape, t.stride()) and t.data_ptr() % 16 == 0):
        return t
    import torch
    return t.clone(memory_format=torch.contiguous_format)


def _autograd_function():
    import torch

    class RotaryFunction(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, positions, rot, inverse):
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(positions)
            ctx.rot, ctx.inverse = rot, inverse
            return rotary_fwd(_dense(q), None if k is None else _dense(k), positions, rot, inverse=inverse)

        @staticmethod
        def backward(ctx, dq, dk):
            # a rotation's gradient is the rotation back, of the queries' and
            # the keys' gradients in one launch where both came; itself
            # differentiable where the backward pass is recorded
            positions, = ctx.saved_tensors
            need_q, need_k = ctx.needs_input_grad[:2]
            if not need_q:
                dq = None
            if not need_k:
                dk = None
            if dq is None and dk is None:
                return None, None, None, None, None
            a, b = (dq, dk) if dq is not None else (dk, None)
            if torch.is_grad_enabled():
                a, b = RotaryFunction.apply(a, b, positions, ctx.rot, not ctx.inverse)
            else:
                a, b = rotary_fwd(_dense(a), None if b is None else _dense(b), positions, ctx.rot, inverse=not ctx.inverse)
            return (a, b, None, None, None) if dq is not None else (None, a, None, None, None)
    return RotaryFunction


def _has_tangent(forward_ad, *tensors) -> bool:
    """Whether one of them is a dual tensor of forward-mode differentiation."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


_ROTARY_FN = None


def rotary(q, k, positions, rot: Rotary):
    """rotary_fwd, differentiable in q and k (either may need no gradient; k
    may be None): both rotations are one launch of gr_rotary, and so are their
    gradients. Forward-mode tangents are refused (NotImplementedError), as by
    flash_attention. A backward pass captured into a graph takes
    torch.autograd.grad: an eager backward of the same leaves on another stream,
    still alive, must not be joined by a captured one (torch's own rule)."""
    import torch
    recorded = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
    forward_ad = torch.autograd.forward_ad
    if not recorded and (forward_ad._current_level < 0 or not _has_tangent(forward_ad, q, k)):
        return rotary_fwd(_dense(q), None if k is None else _dense(k), positions, rot)
    global _ROTARY_FN
    if _ROTARY_FN is None:
        _ROTARY_FN = _autograd_function()
    return _ROTARY_FN.apply(q, k, positions, rot, False)
