"""Python face of the norm of query and key heads that goes before their
rotation (gr_norm_rotary and its gradient).

A head row x becomes x / sqrt(mean(x^2) + eps) times its weights, and is then
turned by its position as by `rotary`: `norm_rotary` does both in one pass,
differentiably in q, k and the weights. `HeadNorm` holds the weights, and
`paged_append` takes one too, for tokens on their way into a cache. The reference has no norm of
heads; its attention (run_attention_search.py:34-114) is what the rows go to.

There is no CPU path: CPU tensors or a missing library raise.
"""
from __future__ import annotations

import ctypes
import functools

from . import runtime as rt
from .rotary import (Rotary, _dense, _has_tangent, _tokens, check_out, check_positions, head_strides)


class HeadNorm:
    """The norm of heads: q_weight and k_weight are contiguous [head_dim] tensors on
    the GPU, at 16-byte aligned addresses, both in float32 or both in the heads' dtype,
    or None for no weights; eps is added to the mean square (with 0, a row of zeros is
    NaN, and rows are normed from magnitudes of 2^-60 on: squares of less are lost)."""

    def __init__(self, q_weight=None, k_weight=None, eps: float = 1e-6):
        if not 0.0 <= eps < 1e30:
            raise ValueError(f"HeadNorm: eps {eps} must not be negative")
        self.q_weight, self.k_weight, self.eps = q_weight, k_weight, float(eps)

    def spec(self, head_dim: int, dtype, index: int, who: str):
        """The gr_head_norm of the weights as they are now, for heads of `dtype` on GPU `index`."""
        return _spec(self.q_weight, self.k_weight, self.eps, head_dim, dtype, index, who)


def _spec(q, k, eps, head_dim, dtype, index, who):
    """The gr_head_norm of weights q and k (or None), checked."""
    of = dtype
    for w in (q, k):
        if w is None:
            continue
        if w.dim() != 1 or w.numel() != head_dim or w.get_device() != index or not w.is_contiguous():
            raise ValueError(f"{who}: the norm's weights must be contiguous [{head_dim}] tensors on GPU {index}, not "
                             f"{tuple(w.shape)} on {w.device}")
        of = w.dtype
    code = rt.dtype_code(of)
    if (code != rt.GR_F32 and of != dtype) or (q is not None and q.dtype != of):
        raise ValueError(f"{who}: the norm's weights must both be float32 or {dtype}")
    return rt.HeadNormSpec(None if q is None else q.data_ptr(), None if k is None else k.data_ptr(), code, eps)


@functools.lru_cache(maxsize=4096)
def _bwd_workspace(index, *sizes):
    """Bytes of a call on GPU `index`, whose compute units share it out."""
    import torch
    with torch.cuda.device(index):
        return int(rt.lib().gr_norm_rotary_bwd_workspace(*sizes))


def _sizes(q, k, rot, who):
    """_tokens of checked q and k."""
    if q is None:
        raise ValueError(f"{who}: q must be given")
    ok = rot.index >= 0 and q.get_device() == rot.index
    if k is None:
        sizes = _tokens(q.shape, q.stride(), None, None, rot.head_dim)
    else:
        sizes = _tokens(q.shape, q.stride(), k.shape, k.stride(), rot.head_dim)
        ok = ok and k.get_device() == rot.index and k.dtype == q.dtype
    if sizes is None or not ok:
        raise ValueError(f"{who}: q and k must be [B, H, N, {rot.head_dim}] tensors of one dtype, B and N on {rot.device} "
                         "(no CPU path) with unit stride on their last dimension")
    if sizes == "too many":
        raise ValueError(f"{who}: {tuple(q.shape)} is too many tokens or heads for one call (2^31)")
    return sizes


def norm_rotary_fwd(q, k, positions, rot: Rotary, norm: HeadNorm, *, out=None, k_out=None, stream=None):
    """rotary_fwd of normed heads: q [B, Hq, N, D] and k [B, Hk, N, D] (or None),
    fp16, bf16 or fp32, each row normed by `norm` in fp32 (magnitudes up to 2^59,
    beyond which the squares' sum is no fp32 number) and turned to its position; other arguments, and what is returned, as
    rotary_fwd's."""
    who = "norm_rotary"
    B, N, Hq, qs, Hk, ks = _sizes(q, k, rot, who)
    ps = check_positions(positions, rot, (B, N), who)
    spec = norm.spec(rot.head_dim, q.dtype, rot.index, who)
    out = check_out(out, q, "out", who, stream)
    head = (rot.ref, ctypes.addressof(spec), q.data_ptr(), out.data_ptr(), Hq, qs, head_strides(out, "out", who))
    if k is None:
        head += (None, None, 0, None, None)
    else:
        k_out = check_out(k_out, k, "k_out", who, stream)
        k_to = k_out.data_ptr()
        if k_to == head[3] and k_to:
            raise ValueError(f"{who}: `out` and `k_out` must be two tensors")
        head += (k.data_ptr(), k_to, Hk, ks, head_strides(k_out, "k_out", who))
    if B == 0 or N == 0:
        return out, k_out
    rt.launch(rt.lib().gr_norm_rotary, head + (rt.dtype_code(q.dtype), B, N, positions.data_ptr(), ps), q, stream,
              "gr_norm_rotary")
    return out, k_out


def norm_rotary_bwd(q, k, positions, rot: Rotary, norm: HeadNorm, dq_out, dk_out, *, weights: bool = True, stream=None):
    """The gradient of norm_rotary_fwd: from its q and k (or None) and the
    gradients of its results, (dq, dk, dq_weight, dk_weight), new tensors laid out as
    dq_out, dk_out and the weights; None for what there is none of, and the weights' with
    weights=False. The weights' gradients are summed in fp32, in an order that the sizes alone
    decide."""
    return _bwd(q, k, positions, rot, norm.q_weight, norm.k_weight, norm.eps, dq_out, dk_out, weights, weights, stream)


def _bwd(q, k, positions, rot, q_weight, k_weight, eps, dq_out, dk_out, want_q, want_k, stream=None):
    """norm_rotary_bwd; want_q, want_k: the weights whose gradients are wanted."""
    who = "norm_rotary_bwd"
    B, N, Hq, qs, Hk, ks = _sizes(q, k, rot, who)
    ps = check_positions(positions, rot, (B, N), who)
    spec = _spec(q_weight, k_weight, eps, rot.head_dim, q.dtype, rot.index, who)
    for name, g, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        if (g is None) != (x is None) or (g is not None and (g.shape != x.shape or g.dtype != x.dtype or g.device != x.device)):
            raise ValueError(f"{who}: {name} must be as its heads, {None if x is None else tuple(x.shape)}")
    outs = [rt.empty_like(g, stream) if g is not None else None for g in (dq_out, dk_out)]
    dws = [rt.empty_like(w, stream) if want and w is not None and x is not None else None
           for w, x, want in ((q_weight, q, want_q), (k_weight, k, want_k))]
    if B == 0 or N == 0:
        import torch
        with torch.cuda.stream(torch.cuda.current_stream(q.device) if stream is None else rt.torch_stream(stream, q.device)):
            return (*outs, *(None if w is None else w.zero_() for w in dws))
    code = rt.dtype_code(q.dtype)
    need = 0 if dws[0] is None and dws[1] is None else _bwd_workspace(rot.index, Hq, Hk, rot.head_dim, B, N)
    ws = rt.workspace(need, q.device, stream) if need else None

    def side(x, g, d, H, st):
        if x is None:
            return (None, None, None, 0, None, None, None)
        return (x.data_ptr(), g.data_ptr(), d.data_ptr(), H, st, head_strides(g, "the gradient", who), head_strides(d, "the gradient", who))
    args = (rot.ref, ctypes.addressof(spec)) + side(q, dq_out, outs[0], Hq, qs) + side(k, dk_out, outs[1], Hk, ks)
    args += (code, B, N, positions.data_ptr(), ps) + tuple(None if w is None else w.data_ptr() for w in dws)
    rt.launch(rt.lib().gr_norm_rotary_bwd, args + (None if ws is None else ws.data_ptr(), need), q, stream, "gr_norm_rotary_bwd")
    return (*outs, *dws)


def _autograd_function():
    import torch

    class NormRotaryFunction(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, q_weight, k_weight, positions, rot, eps):
            ctx.set_materialize_grads(False)
            q, k = _dense(q), None if k is None else _dense(k)
            ctx.save_for_backward(q, k, q_weight, k_weight, positions)
            ctx.rot, ctx.eps = rot, eps
            return norm_rotary_fwd(q, k, positions, rot, HeadNorm(q_weight, k_weight, eps))

        @staticmethod
        def backward(ctx, dq, dk):
            # differentiable once: only where the backward pass is recorded does that
            # have to be kept track of
            return recorded(ctx, dq, dk) if torch.is_grad_enabled() else gradients(ctx, dq, dk)

    def gradients(ctx, dq, dk):
        # queries and keys in one launch where the gradients of both came and are of use
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        need_q, need_k, want_q, want_k = ctx.needs_input_grad[:4]
        if not (need_q or want_q):
            dq = None
        if not (need_k or want_k):
            dk = None
        if dq is None and dk is None:
            return (None,) * 7
        if dq is None:                                         # keys alone, as the queries of a call
            g, _, w, _ = _bwd(k, None, positions, ctx.rot, k_weight, None, ctx.eps, _dense(dk), None, want_k, False)
            return None, g, None, w, None, None, None
        if dk is None:
            g, _, w, _ = _bwd(q, None, positions, ctx.rot, q_weight, None, ctx.eps, _dense(dq), None, want_q, False)
            return g, None, w, None, None, None, None
        return (*_bwd(q, k, positions, ctx.rot, q_weight, k_weight, ctx.eps, _dense(dq), _dense(dk), want_q, want_k),
                None, None, None)
    recorded = torch.autograd.function.once_differentiable(gradients)
    return NormRotaryFunction


_NORM_ROTARY_FN = None


def norm_rotary(q, k, positions, rot: Rotary, norm: HeadNorm):
    """norm_rotary_fwd, differentiable once in q, k (which may be None) and the
    weights: both are one launch, and so are their gradients, with a second one that adds
    up the weights'. Forward-mode tangents are refused (NotImplementedError), as by
    rotary, whose rule for a backward pass captured into a graph holds here too."""
    import torch
    w, v = norm.q_weight, norm.k_weight
    recorded = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, w, v))
    forward_ad = torch.autograd.forward_ad
    if not recorded and (forward_ad._current_level < 0 or not _has_tangent(forward_ad, q, k, w, v)):
        return norm_rotary_fwd(_dense(q), None if k is None else _dense(k), positions, rot, norm)
    global _NORM_ROTARY_FN
    if _NORM_ROTARY_FN is None:
        _NORM_ROTARY_FN = _autograd_function()
    return _NORM_ROTARY_FN.apply(q, k, w, v, positions, rot, norm.eps)
