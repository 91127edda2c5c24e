"""Gradients of normed and rotated heads: what queries' and keys' weights share, what is not needed, magnitudes at the
ends of the range, and calls whose waves walk over several tokens."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_norm_gpu import (BWD, FWD, _check, _gradients, _inputs, _normed, _size, _turned,  # noqa: E402
                           test_forward as _forward_of, test_gradients as _gradients_of)
from test_rotary_gpu import DT, _cuda  # noqa: E402


@pytest.mark.parametrize("B,N,Hq,Hk,D,rd,dtype,weights", [
    (1, 20, 3, 2, 64, 64, "fp32", "same"),          # all heads in one pass
    (2, 33, 9, 3, 128, 64, "bf16", "fp32"),         # the last query head beside the keys'
    (1, 40, 5, 4, 80, 48, "fp16", "same"),          # lanes without elements
    (1, 700, 17, 2, 64, 32, "fp16", "fp32"),
])
@pytest.mark.parametrize("what", ["x", "gradient"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_that_are_not_finite_reach_their_own_weights_only(B, N, Hq, Hk, D, rd, dtype, weights, what, value):
    """Queries and keys that one pass works on: a query's NaN or infinity is in no sum of the keys' weights, nor a key's
    in the queries'."""
    dev = _cuda()
    from grammar.norm import norm_rotary_bwd
    print(f"[case] weights B{B} N{N} H{Hq}/{Hk} D{D}/{rd} {dtype} {weights} {what} {value}", flush=True)
    g, rot, norm, q, k, pos = _inputs(B, N, Hq, Hk, D, rd, None, False, dtype, weights, dev)
    dq, dk = (torch.randn(t.shape, generator=g).to(t.dtype).to(dev) for t in (q, k))
    want = norm_rotary_bwd(q, k, pos, rot, norm, dq, dk)
    assert all(t.isfinite().all() for t in want[2:])
    for i, (x, dy) in enumerate(((q, dq), (k, dk))):
        to = x if what == "x" else dy
        keep = to.clone()
        to[B - 1, -1 if i == 0 else 0, N // 2, 5] = value
        got = norm_rotary_bwd(q, k, pos, rot, norm, dq, dk)
        to.copy_(keep)
        assert torch.equal(got[3 - i], want[3 - i]) and torch.equal(got[1 - i], want[1 - i])
        assert not got[2 + i].isfinite().all()


@pytest.mark.parametrize("frozen", ["q", "k"])
@pytest.mark.parametrize("weights", [None, "frozen", "trained"])
def test_a_side_without_gradients_is_left_out(frozen, weights, monkeypatch):
    """Queries or keys that need no gradient, nor do their weights: the backward pass does not read or write them."""
    dev = _cuda()
    from grammar import norm as gn
    from grammar.rotary import Rotary
    rot, pos = Rotary(64, device=dev), torch.arange(40, dtype=torch.int32, device=dev)
    q, k = torch.randn((2, 6, 40, 64), device=dev).bfloat16(), torch.randn((2, 2, 40, 64), device=dev).bfloat16()
    leaf = (k if frozen == "q" else q).requires_grad_()
    w = [None, None] if weights is None else [1 + 0.2 * torch.randn(64, device=dev) for _ in range(2)]
    if weights == "trained":                                        # the other side's
        w[frozen == "q"].requires_grad_()
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    calls, bwd = [], gn._bwd
    monkeypatch.setattr(gn, "_bwd", lambda *a, **kw: (calls.append(a[:2]), bwd(*a, **kw))[1])
    wanted = [leaf] + [t for t in w if t is not None and t.requires_grad]
    got = torch.autograd.grad(gn.norm_rotary(q, k, pos, rot, gn.HeadNorm(*w)), wanted, (dq, dk))
    assert [tuple(None if t is None else t.data_ptr() for t in c) for c in calls] == [(leaf.data_ptr(), None)]
    mine, g = (w[1], dk) if frozen == "q" else (w[0], dq)
    want = bwd(leaf.detach(), None, pos, rot, None if mine is None else mine.detach(), None, 1e-6, g, None, weights == "trained", False)
    assert torch.equal(got[0], want[0])
    assert len(got) == 1 or torch.equal(got[1], want[2])


@pytest.mark.parametrize("D,dtype,weights", [(256, "fp32", "same"), (256, "bf16", "fp32"), (128, "bf16", "same"), (64, "fp32", None)])
@pytest.mark.parametrize("power,eps", [(59, 1e-6), (59, 0.0), (-60, 0.0), (-60, 1e-6)])
def test_magnitudes_at_the_ends_of_the_range(D, dtype, weights, power, eps):
    """Rows of magnitudes up to 2^59, one of them that number throughout (256 squares of 2^60 are no fp32 number), and,
    without eps, from 2^-60 on: forward and gradient."""
    dev = _cuda()
    from grammar.norm import HeadNorm, norm_rotary_bwd, norm_rotary_fwd
    print(f"[case] ends D{D} {dtype} {weights} 2^{power} eps {eps}", flush=True)
    g, rot, norm, q, k, pos = _inputs(2, 19, 5, 2, D, D, None, False, dtype, weights, dev)
    q, k = ((torch.rand(t.shape, generator=g) + 1) * 2.0 ** (power - 1) * (torch.randint(0, 2, t.shape, generator=g) * 2 - 1) for t in (q, k))
    q[1, 2, 3], k[0, 1, 4] = 2.0 ** power, -2.0 ** power
    q, k = q.to(DT[dtype]).to(dev), k.to(DT[dtype]).to(dev)
    assert q.abs().max() == 2.0 ** power and k.abs().max() == 2.0 ** power
    norm = HeadNorm(norm.q_weight, norm.k_weight, eps)
    got = norm_rotary_fwd(q, k, pos, rot, norm)
    dq, dk = (torch.randn(t.shape, generator=g).to(t.dtype).to(dev) for t in (q, k))
    back = norm_rotary_bwd(q, k, pos, rot, norm, dq, dk)
    for i, (x, dy, w) in enumerate(((q, dq, norm.q_weight), (k, dk, norm.k_weight))):
        y, size = _turned(_normed(x, w, eps)[0], pos, rot)
        _check(got[i], y, _size(y, size), "rows", FWD)
        dx, dw, xs, ws = _gradients(x, dy, w, pos, rot, eps)
        _check(back[i], dx, xs, "gradient", BWD)
        if w is not None:
            _check(back[2 + i], dw, ws, "weights' gradient", 100 * 2.0 ** -24)


@pytest.mark.parametrize("B,N,Hq,Hk,D,rd,sections,inter,dtype,weights", [
    (3, 1571, 16, 16, 64, 64, [10, 11, 11], True, "fp16", "fp32"),
    (2, 4096, 32, 8, 128, 128, None, False, "bf16", "same"),
    (1, 4111, 9, 3, 128, 64, [12, 20], False, "fp32", "same"),
    (2, 2081, 20, 6, 96, 96, [16, 16, 16], False, "bf16", "fp32"),     # lanes without elements, in every pass
    (1, 4300, 33, 1, 80, 48, None, True, "fp32", "same"),
    (4, 1100, 7, 7, 240, 128, [32, 0, 32], False, "fp16", "fp32"),
    (1, 9001, 6, 2, 64, 32, [8, 8], True, "bf16", "same"),             # one pass a token, five tokens a wave
    (1, 13_007, 12, 4, 64, 64, [16, 16], False, "fp32", None),
])
def test_waves_that_walk_over_tokens(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights):
    """From 4,096 tokens on, 2 for each wave of 256 compute units, a wave takes all passes of a token and then another's:
    rows and positions of the next one are asked for ahead, over the end of a token and of a sequence. (Sums of the
    weights' gradients: at most 20 rows a lane, 4 additions over lanes, 4 over waves and 14 over workgroups.)"""
    _gradients_of(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights)
    _forward_of(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights)
