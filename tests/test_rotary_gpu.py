"""Position rotation (gr_rotary) against the formula in 64 bits: layouts, axes,
types, sizes, far and negative positions, gradients, streams and graphs."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def _exact(x, pos, rot, sign=1):
    """x [B, H, N, D] rotated in 64 bits, and per element |x1| + |x2| of its pair."""
    rd, pairs = rot.rotary_dim, rot.rotary_dim // 2
    freq = torch.tensor(rot.inv_freq, dtype=torch.float64, device=x.device)
    p = pos.double() if rot.naxes > 1 else pos.double()[None]
    axis = torch.tensor([a for a, n in enumerate(rot.sections) for _ in range(n)], device=x.device)
    ang = sign * p[axis].movedim(0, -1) * freq                    # [N, pairs] or [B, N, pairs]
    if ang.dim() == 3:
        ang = ang[:, None]
    x = x.double()
    i, j = (torch.arange(0, rd, 2), torch.arange(1, rd, 2)) if rot.interleaved else (torch.arange(pairs), torch.arange(pairs, rd))
    a, b = x[..., i], x[..., j]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = a * torch.cos(ang) - b * torch.sin(ang), a * torch.sin(ang) + b * torch.cos(ang)
    size[..., i] = size[..., j] = a.abs() + b.abs()
    return y, size


def _check(got, want, size, what):
    """One rounding to the type (half a step; fp16 below 2^-14 half of 2^-24),
    and fp32 arithmetic: the angle's three roundings (3 2^-24 of pi / 4), the
    sums of sine and cosine (2^-23), two products and a sum (2^-23), each of
    |x1| + |x2|: 4e-7 together."""
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 4e-7 * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    bad = (got.double() - want).abs() > tol * (1 + 1e-6)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() - tol).max())}"


CASES = [
    # B, N, Hq, Hk, D, rotary_dim, sections, per_axis, interleaved, dtype
    (1, 1, 1, 1, 64, 64, None, False, False, "bf16"),
    (2, 33, 8, 2, 128, 128, None, False, False, "bf16"),
    (2, 33, 8, 2, 128, 128, None, False, True, "fp16"),
    (3, 130, 5, 1, 64, 32, [5, 5, 6], False, False, "fp16"),
    (1, 257, 3, 3, 128, 128, [16, 24, 24], False, False, "bf16"),
    (2, 64, 16, 16, 64, 64, [10, 11, 11], True, True, "fp32"),
    (1, 19, 2, 2, 80, 48, [24, 0], True, False, "fp32"),
    (1, 7, 4, 1, 256, 256, [16] * 8, False, False, "bf16"),
    (4, 1000, 12, 4, 96, 96, None, False, False, "fp32"),
    (2, 2048, 32, 8, 128, 64, None, False, True, "bf16"),
    # several passes of a wave, the last one part-filled; stores of whole lines and of parts
    (2, 701, 33, 8, 128, 128, None, False, False, "bf16"),
    (1, 700, 13, 6, 256, 128, None, False, False, "fp16"),
    (3, 900, 25, 12, 64, 32, None, False, False, "fp16"),
    (1, 1500, 17, 3, 128, 96, [20, 28], False, False, "fp32"),
]


@pytest.mark.parametrize("B,N,Hq,Hk,D,rd,sections,per_axis,inter,dtype", CASES)
def test_rotary_matches_the_formula(B, N, Hq, Hk, D, rd, sections, per_axis, inter, dtype):
    dev = _cuda()
    from grammar.rotary import Rotary, rotary_fwd
    print(f"[case] rotary B{B} N{N} H{Hq}/{Hk} D{D}/{rd} {sections} {dtype}", flush=True)
    g = torch.Generator("cpu").manual_seed(N + D)
    rot = Rotary(D, rotary_dim=rd, sections=sections, per_axis=per_axis, interleaved=inter, device=dev)
    q, k = (torch.randn((B, h, N, D), generator=g).to(DT[dtype]).to(dev) for h in (Hq, Hk))
    lead = (rot.naxes,) if rot.naxes > 1 else ()
    for shape in ((N,), (B, N)):
        pos = torch.randint(-500, 300_000, lead + shape, generator=g, dtype=torch.int32).to(dev)
        for inverse in (False, True):
            qo, ko = rotary_fwd(q, k, pos, rot, inverse=inverse)
            assert qo.dtype == q.dtype and qo.shape == q.shape
            for got, x, name in ((qo, q, "q"), (ko, k, "k")):
                _check(got, *_exact(x, pos, rot, -1 if inverse else 1), f"{name} {shape} inverse={inverse}")
        only, none = rotary_fwd(q, None, pos, rot)
        assert none is None and torch.equal(only, rotary_fwd(q, k, pos, rot)[0])


def test_far_positions_keep_their_angle():
    dev = _cuda()
    from grammar.rotary import Rotary, rotary_fwd
    rot = Rotary(64, device=dev)
    q = torch.randn((1, 2, 6, 64), device=dev)
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 10 ** 9, -(10 ** 9), 2 ** 24 + 1, 0], dtype=torch.int32, device=dev)
    # the oracle's own angle is off by 2^-53 of up to 2^31 radians, 2.4e-7
    want, size = _exact(q, pos, rot)
    got = rotary_fwd(q, None, pos, rot)[0]
    assert ((got.double() - want).abs() <= 2.0 ** -24 * want.abs() + 8e-7 * size).all()


def test_strided_heads_in_place_and_layout():
    dev = _cuda()
    from grammar.rotary import Rotary, rotary_fwd
    rot = Rotary(128, rotary_dim=64, device=dev)
    rows = torch.randn((2, 45, 14, 128), device=dev).bfloat16()       # a projection's rows: 8 q, 2 k heads, the rest
    q, k = rows[:, :, :8].transpose(1, 2), rows[:, :, 8:10].transpose(1, 2)
    pos = torch.arange(45, dtype=torch.int32, device=dev)
    want_q, want_k = (_exact(t, pos, rot) for t in (q, k))
    keep = rows.clone()
    qo, ko = rotary_fwd(q, k, pos, rot)
    assert torch.equal(rows, keep)
    assert qo.stride(1) < qo.stride(2)                                # laid out as q: heads inside tokens
    _check(qo, *want_q, "q")
    _check(ko, *want_k, "k")
    rotary_fwd(q, k, pos, rot, out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(rows[:, :, 10:], keep[:, :, 10:])              # the neighbours are untouched


def test_values_that_do_not_turn_pass_unchanged():
    dev = _cuda()
    from grammar.rotary import Rotary, rotary_fwd
    rot = Rotary(64, rotary_dim=32, device=dev)
    q = torch.full((1, 1, 3, 64), float("inf"), device=dev, dtype=torch.float16)
    q[..., :32] = 1.0
    q[0, 0, 1, 40] = float("nan")
    pos = torch.arange(3, dtype=torch.int32, device=dev)
    got = rotary_fwd(q, None, pos, rot)[0]
    assert torch.equal(got[..., 32:].view(torch.int16), q[..., 32:].view(torch.int16))
    assert got[..., :32].isfinite().all()


@pytest.mark.parametrize("inter,sections", [(False, None), (True, [3, 5, 8])])
def test_gradients_against_formula_and_differences(inter, sections):
    dev = _cuda()
    from grammar.rotary import Rotary, rotary
    rot = Rotary(48, rotary_dim=32, interleaved=inter, sections=sections, device=dev)
    g = torch.Generator("cpu").manual_seed(5)
    q = torch.randn((2, 3, 5, 48), generator=g).to(dev).requires_grad_()
    k = torch.randn((2, 1, 5, 48), generator=g).to(dev).requires_grad_()
    pos = torch.randint(0, 90, ((rot.naxes,) if rot.naxes > 1 else ()) + (5,), generator=g, dtype=torch.int32).to(dev)
    wq, wk = torch.randn(q.shape, generator=g).to(dev), torch.randn(k.shape, generator=g).to(dev)
    qo, ko = rotary(q, k, pos, rot)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (wq, wk))
    _check(dq, *_exact(wq, pos, rot, -1), "dq")
    _check(dk, *_exact(wk, pos, rot, -1), "dk")
    # a difference along a direction: the loss is linear, so its step may be 1
    with torch.no_grad():
        d = torch.randn(q.shape, generator=g).to(dev)
        up, down = (float((rotary(q + s * d, k, pos, rot)[0].double() * wq.double()).sum()) for s in (1.0, -1.0))
    want = float((dq.double() * d.double()).sum())
    assert abs((up - down) / 2 - want) <= 1e-5 * float((dq.double() * d.double()).abs().sum())


def test_broadcast_missing_and_partial_gradients():
    dev = _cuda()
    from grammar.rotary import Rotary, rotary
    rot = Rotary(64, device=dev)
    pos = torch.arange(9, dtype=torch.int32, device=dev)
    q = torch.randn((2, 4, 9, 64), device=dev).bfloat16().requires_grad_()
    k = torch.randn((2, 4, 9, 64), device=dev).bfloat16()
    qo, ko = rotary(q, k, pos, rot)
    qo.sum().backward()                                               # a gradient with strides of zero
    ones = torch.ones_like(q)
    _check(q.grad, *_exact(ones, pos, rot, -1), "dq of a sum")
    assert k.grad is None
    k = k.clone().requires_grad_()
    qo, ko = rotary(q.detach(), k, pos, rot)
    ko[..., 1::2].sum().backward()                                    # only the keys' output is used
    one = torch.zeros_like(k)
    one[..., 1::2] = 1
    _check(k.grad, *_exact(one, pos, rot, -1), "dk of a slice")
    q1 = torch.randn((1, 4, 9, 64), device=dev).bfloat16().requires_grad_()
    qo, _ = rotary(q1.expand(3, 4, 9, 64), None, pos, rot)            # a broadcast input: its gradient is the sum
    qo.backward(torch.ones_like(qo))
    one = _exact(torch.ones_like(q1), pos, rot, -1)[0]
    # three equal bf16 gradients, added in bf16: each and the sums round once
    assert ((q1.grad.double() - 3 * one).abs() <= 3 * 2.0 ** -8 * 3 * one.abs() + 1e-5).all()


def test_gradient_of_the_gradient():
    """The gradient is linear in the one that comes in: differentiated again it is the forward rotation."""
    dev = _cuda()
    from grammar.rotary import Rotary, rotary
    rot = Rotary(32, device=dev)
    pos = torch.arange(5, dtype=torch.int32, device=dev)
    q, k, w = (torch.randn((1, 2, 5, 32), device=dev).requires_grad_() for _ in range(3))
    qo, ko = rotary(q, k, pos, rot)
    dq, dk = torch.autograd.grad((qo * w).sum() + ko.sum(), (q, k), create_graph=True)
    u = torch.randn_like(q)
    dw, = torch.autograd.grad(dq, w, u)
    _check(dw, *_exact(u, pos, rot), "d dq / d w")


def test_rotated_training_attention_gradients():
    """rotary and flash_attention as a training step runs them, against 64 bits."""
    dev = _cuda()
    from grammar.attention import flash_attention
    from grammar.rotary import Rotary, rotary
    B, H, N, D = 1, 2, 128, 64
    rot = Rotary(D, device=dev)
    pos = torch.arange(N, dtype=torch.int32, device=dev)
    g = torch.Generator("cpu").manual_seed(11)
    q, k, v, do = (torch.randn((B, H, N, D), generator=g).half().to(dev) for _ in range(4))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    qr, kr = rotary(leaves[0], leaves[1], pos, rot)
    o = flash_attention(qr, kr, leaves[2], causal=True)
    grads = torch.autograd.grad(o, leaves, do)
    ref = [t.double().clone().requires_grad_() for t in (q, k, v)]
    rq, rk = (_exact(t, pos, rot)[0] for t in ref[:2])
    s = (rq @ rk.transpose(2, 3).contiguous()) / math.sqrt(D)
    s = s.masked_fill(torch.ones(N, N, dtype=torch.bool, device=dev).triu(1), float("-inf"))
    ro = torch.softmax(s, -1) @ ref[2]
    want = torch.autograd.grad(ro, ref, do.double())
    # fp16 rounds q and k once more than the oracle (2^-11 of scores up to 6 or
    # so), then P, dS and the results: a few 2^-11 of the largest entry
    for got, w in zip((o, *grads), (ro, *want)):
        assert (got.double() - w).detach().abs().max() <= 8 * 2.0 ** -11 * max(1.0, float(w.detach().abs().max()))


def test_other_streams_and_graph_replays():
    dev = _cuda()
    from grammar.rotary import Rotary, rotary, rotary_fwd
    rot = Rotary(128, device=dev)
    q, k = (torch.randn((1, h, 77, 128), device=dev).bfloat16() for h in (6, 2))
    pos = torch.arange(77, dtype=torch.int32, device=dev)
    want = rotary_fwd(q, k, pos, rot)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        out = [torch.zeros_like(t) for t in want]
        side.wait_stream(torch.cuda.current_stream())
        rotary_fwd(q, k, pos, rot, out=out[0], k_out=out[1], stream=stream)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    leaf = q.clone().requires_grad_()
    with torch.cuda.stream(side):
        rotary(leaf, k, pos, rot)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            qo, ko = rotary(leaf, k, pos, rot)
            dq, = torch.autograd.grad(qo, leaf, qo.detach())
    torch.cuda.synchronize()
    for i in range(4):
        with torch.no_grad():
            leaf.copy_(torch.randn_like(leaf))
            pos.add_(i * 1000)
        graph.replay()
        torch.cuda.synchronize()
        a, b = rotary_fwd(leaf.detach(), k, pos, rot)
        assert torch.equal(qo, a) and torch.equal(ko, b)
        assert torch.equal(dq, rotary_fwd(a, None, pos, rot, inverse=True)[0])


def test_refusals():
    dev = _cuda()
    from grammar import runtime as rt
    from grammar.rotary import Rotary, rotary_fwd
    rot, two = Rotary(64, device=dev), Rotary(64, sections=[16, 16], device=dev)
    q, pos = torch.randn((1, 2, 8, 64), device=dev).half(), torch.arange(8, dtype=torch.int32, device=dev)
    for bad in (lambda: rotary_fwd(q.cpu(), None, pos, rot), lambda: rotary_fwd(q, None, pos.long(), rot),
                lambda: rotary_fwd(q, None, pos[:7], rot), lambda: rotary_fwd(q, None, pos, two),
                lambda: rotary_fwd(q, q.float(), pos, rot), lambda: rotary_fwd(q, q[:, :, :4], pos, rot),
                lambda: rotary_fwd(q[..., :32], None, pos, rot), lambda: rotary_fwd(None, q, pos, rot),
                lambda: rotary_fwd(q, None, pos, rot, out=q[:, :1]), lambda: rotary_fwd(q, None, pos.cpu(), rot),
                lambda: rotary_fwd(q.transpose(2, 3).contiguous().transpose(2, 3), None, pos, rot),
                lambda: rotary_fwd(q.double(), None, pos, rot)):
        with pytest.raises(ValueError):
            bad()
    on_cpu = Rotary(64, device="cpu")
    with pytest.raises(ValueError, match="GPU|CPU"):
        rotary_fwd(q.cpu(), None, pos.cpu(), on_cpu)
    with pytest.raises(ValueError):
        rotary_fwd(q, None, pos, rot, out=q[:, :1].expand(1, 2, 8, 64))
    to = torch.empty_like(q)
    with pytest.raises(ValueError, match="two tensors"):
        rotary_fwd(q, q, pos, rot, out=to, k_out=to)
    odd = torch.randn(1 * 2 * 8 * 64 + 4, device=dev).half()[4:].view(1, 2, 8, 64)
    with pytest.raises(rt.GrError, match="aligned"):
        rotary_fwd(odd, None, pos, rot)
    wide = torch.randn((1, 2, 8, 68), device=dev).half()[..., :64]
    with pytest.raises(rt.GrError, match="multiples of 8"):
        rotary_fwd(wide, None, pos, rot)
    assert rotary_fwd(q[:, :, :0], None, pos[:0], rot)[0].shape == (1, 2, 0, 64)
