"""Normed and rotated heads (gr_norm_rotary) and their gradient against the formula
in 64 bits: layouts, types, sizes, weights, strides, streams and graphs."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_rotary_gpu import DT, _cuda, _exact as _turned  # noqa: E402


def _normed(x, w, eps):
    """(normed rows, 1 / sqrt(mean x^2 + eps)) in 64 bits."""
    x = x.double()
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r * (1.0 if w is None else w.double()), r


def _size(y, size):
    """|y1| + |y2| of a turned pair, |y| of an element that does not turn."""
    return torch.where(size > 0, size, y.abs())


def _check(got, want, size, what, coef):
    """One rounding to the type (half a step; fp16 below 2^-14 half of 2^-24) and coef of `size` for the fp32
    arithmetic before it."""
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() * 1.001 + coef * size + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() - tol).max())}"


# Forward: the sum of D squares adds within 16 elements and over at most 16 lanes, each sum of positive terms (20 2^-24),
# mean, eps and root 4 more, the root halves what was before it: 14; two products 2: 16 2^-24 = 1e-6. The rotation 4e-7.
FWD = 1.4e-6
# Gradient: g turned back 4e-7; r to the third power 3 14, the dot product of D signed terms 20 of their sizes'
# sum, products and the last sum 6: 68 2^-24 = 4.1e-6.
BWD = 4.5e-6


def _weights(kind, D, dtype, g, dev):
    if kind is None:
        return None, None
    t = torch.float32 if kind == "fp32" else DT[dtype]
    return tuple((1 + 0.3 * torch.randn(D, generator=g)).to(t).to(dev) for _ in range(2))


CASES = [
    # B, N, Hq, Hk, D, rotary_dim, sections, interleaved, dtype, weights
    (1, 1, 1, 1, 64, 64, None, False, "bf16", "same"),
    (2, 33, 8, 2, 128, 128, None, False, "bf16", "fp32"),
    (2, 33, 8, 2, 128, 128, None, True, "fp16", "same"),
    (3, 130, 5, 1, 64, 32, [5, 5, 6], False, "fp16", "fp32"),
    (1, 257, 3, 3, 128, 128, [16, 24, 24], False, "bf16", None),
    (2, 64, 16, 16, 64, 64, [10, 11, 11], True, "fp32", "same"),
    (1, 19, 2, 2, 80, 48, [24, 0], False, "fp32", "same"),        # rows of 5, 6 and 3 units: lanes without elements
    (2, 77, 7, 2, 96, 96, None, True, "bf16", "same"),
    (1, 40, 9, 3, 48, 32, None, False, "fp16", "same"),
    (1, 21, 3, 1, 16, 16, None, False, "fp32", "fp32"),
    (1, 7, 4, 1, 256, 256, [16] * 8, False, "bf16", "same"),
    (2, 50, 3, 2, 240, 128, None, False, "bf16", "fp32"),
    (2, 700, 32, 8, 128, 64, None, True, "bf16", "same"),
    # several passes of a wave, the last one part-filled; stores of whole lines
    (2, 701, 33, 8, 128, 128, None, False, "bf16", "same"),
    (3, 900, 25, 12, 64, 32, None, False, "fp16", "fp32"),
]


def _inputs(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights, dev):
    from grammar.norm import HeadNorm
    from grammar.rotary import Rotary
    g = torch.Generator("cpu").manual_seed(N + D)
    rot = Rotary(D, rotary_dim=rd, sections=sections, interleaved=inter, device=dev)
    # rows of different magnitudes, and one of zeros
    q, k = ((torch.randn((B, h, N, D), generator=g) * torch.exp2(2 * torch.randn((B, h, N, 1), generator=g))) for h in (Hq, Hk))
    q[0, 0, 0] = 0
    q, k = q.to(DT[dtype]).to(dev), k.to(DT[dtype]).to(dev)
    wq, wk = _weights(weights, D, dtype, g, dev)
    lead = (rot.naxes,) if rot.naxes > 1 else ()
    pos = torch.randint(-500, 300_000, lead + (B, N), generator=g, dtype=torch.int32).to(dev)
    return g, rot, HeadNorm(wq, wk, eps=1e-5), q, k, pos


@pytest.mark.parametrize("B,N,Hq,Hk,D,rd,sections,inter,dtype,weights", CASES)
def test_forward(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights):
    dev = _cuda()
    from grammar.norm import norm_rotary_fwd
    print(f"[case] norm B{B} N{N} H{Hq}/{Hk} D{D}/{rd} {sections} {dtype} {weights}", flush=True)
    g, rot, norm, q, k, pos = _inputs(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights, dev)
    for p in (pos, pos[..., 0, :]):
        qo, ko = norm_rotary_fwd(q, k, p, rot, norm)
        for got, x, w, name in ((qo, q, norm.q_weight, "q"), (ko, k, norm.k_weight, "k")):
            assert got.dtype == x.dtype and got.shape == x.shape
            y, size = _turned(_normed(x, w, norm.eps)[0], p, rot)
            _check(got, y, _size(y, size), name, FWD)
        only, none = norm_rotary_fwd(q, None, p, rot, norm)
        assert none is None and torch.equal(only, qo)
    assert not qo[0, 0, 0].any()


def _gradients(x, dy, w, pos, rot, eps):
    """dx, dw of rows [B, H, N, D] by the formula in 64 bits, and the sizes that their fp32 arithmetic goes by."""
    g, size = _turned(dy, pos, rot, -1)
    size = _size(g, size)
    x = x.double()
    v = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double()
    r = _normed(x, None, eps)[1]
    h, hs = g * v, size * v.abs()
    dx = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
    return dx, (g * x * r).sum((0, 1, 2)), r * (hs + x.abs() * r * r * (hs * x.abs()).mean(-1, keepdim=True)), (size * x.abs() * r).sum((0, 1, 2))


@pytest.mark.parametrize("B,N,Hq,Hk,D,rd,sections,inter,dtype,weights", CASES)
def test_gradients(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights):
    dev = _cuda()
    from grammar.norm import norm_rotary_bwd
    print(f"[case] gradient B{B} N{N} H{Hq}/{Hk} D{D}/{rd} {sections} {dtype} {weights}", flush=True)
    g, rot, norm, q, k, pos = _inputs(B, N, Hq, Hk, D, rd, sections, inter, dtype, weights, dev)
    dq, dk = (torch.randn(t.shape, generator=g).to(t.dtype).to(dev) for t in (q, k))
    got = norm_rotary_bwd(q, k, pos, rot, norm, dq, dk)
    again = norm_rotary_bwd(q, k, pos, rot, norm, dq, dk)
    for i, (x, dy, w, name) in enumerate(((q, dq, norm.q_weight, "q"), (k, dk, norm.k_weight, "k"))):
        dx, dw, xs, ws = _gradients(x, dy, w, pos, rot, norm.eps)
        # a row of zeros has r = 1 / sqrt(1e-5): its gradient in fp16 stays below 65504
        _check(got[i], dx, xs, "d" + name, BWD)
        assert torch.equal(got[i], again[i])
        if w is None:
            assert got[2 + i] is None
            continue
        # g x r as above (32 2^-24 of each), and sums over a wave's rows, its lanes, the waves and the workgroups:
        # at most 60 additions in a chain, each 2^-24 of the sizes' sum at most
        _check(got[2 + i], dw, ws, f"d{name}_weight", 100 * 2.0 ** -24)
        assert got[2 + i].dtype == w.dtype and torch.equal(got[2 + i], again[2 + i])
    alone = norm_rotary_bwd(q, None, pos, rot, norm, dq, None, weights=False)
    assert torch.equal(alone[0], got[0]) and alone[1:] == (None, None, None)


@pytest.mark.parametrize("inter,sections,dtype", [(False, None, "fp32"), (True, [3, 5, 8], "fp32")])
def test_gradients_against_differences(inter, sections, dtype):
    dev = _cuda()
    from grammar.norm import HeadNorm, norm_rotary
    from grammar.rotary import Rotary
    rot = Rotary(48, rotary_dim=32, interleaved=inter, sections=sections, device=dev)
    g = torch.Generator("cpu").manual_seed(5)
    q, k = (torch.randn((2, h, 5, 48), generator=g).to(dev).requires_grad_() for h in (3, 1))
    wq, wk = ((1 + 0.3 * torch.randn(48, generator=g)).to(dev).requires_grad_() for _ in range(2))
    pos = torch.randint(0, 90, ((rot.naxes,) if rot.naxes > 1 else ()) + (5,), generator=g, dtype=torch.int32).to(dev)
    uq, uk = (torch.randn(t.shape, generator=g).to(dev) for t in (q, k))
    leaves = [q, k, wq, wk]
    qo, ko = norm_rotary(q, k, pos, rot, HeadNorm(wq, wk))
    grads = torch.autograd.grad((qo, ko), leaves, (uq, uk))

    def loss(at, exact):
        if exact:
            y = [_turned(_normed(x, w, 1e-6)[0], pos, rot)[0] for x, w in ((at[0], at[2]), (at[1], at[3]))]
        else:
            y = norm_rotary(at[0], at[1], pos, rot, HeadNorm(at[2], at[3]))
        return float((y[0].double() * uq.double()).sum() + (y[1].double() * uk.double()).sum())
    h = 2.0 ** -7
    with torch.no_grad():
        for i in range(4):
            d = torch.randn(leaves[i].shape, generator=g).to(dev)
            ends = [[t + s * h * d if j == i else t for j, t in enumerate(leaves)] for s in (1.0, -1.0)]
            mine, exact = ((loss(ends[0], e) - loss(ends[1], e)) / (2 * h) for e in (False, True))
            slope = float((grads[i].double() * d.double()).sum())
            # what the outputs' roundings (2^-24 and FWD of sizes of at most 4 on average) add to the kernel's difference
            noise = (FWD + 2.0 ** -24) * 4 * (float(uq.abs().sum()) + float(uk.abs().sum())) / h
            assert abs(mine - exact) <= noise, f"leaf {i}"
            # the formula's difference at half the step: what is left of h^2 terms is a quarter there
            ends = [[t + s * h / 2 * d if j == i else t for j, t in enumerate(leaves)] for s in (1.0, -1.0)]
            finer = (loss(ends[0], True) - loss(ends[1], True)) / h
            # (fp32 rounds the steps' ends themselves, 2^-24 of each element, against slopes of the same sizes)
            rounding = 2.0 ** -24 / h * 8 * float((grads[i].double().abs() * (leaves[i].double().abs() + 1)).sum())
            sums = BWD * 40 * float((grads[i].double() * d.double()).abs().sum())
            assert abs(slope - finer) <= abs(exact - finer) + rounding + sums, f"leaf {i}"


def test_partial_broadcast_and_missing_gradients():
    dev = _cuda()
    from grammar.norm import HeadNorm, norm_rotary
    from grammar.rotary import Rotary
    rot = Rotary(64, device=dev)
    pos = torch.arange(9, dtype=torch.int32, device=dev)
    g = torch.Generator("cpu").manual_seed(2)
    q, k = (torch.randn((2, 4, 9, 64), generator=g).bfloat16().to(dev) for _ in range(2))
    wq, wk = ((1 + 0.3 * torch.randn(64, generator=g)).to(dev).requires_grad_() for _ in range(2))
    norm = HeadNorm(wq, wk)
    one = torch.ones_like(q)
    a = q.clone().requires_grad_()
    qo, ko = norm_rotary(a, k, pos, rot, norm)
    qo.sum().backward()                                               # a gradient with strides of zero, keys unused
    dx, dw, xs, ws = _gradients(q, one, wq.detach(), pos, rot, norm.eps)
    _check(a.grad, dx, xs, "dq of a sum", BWD)
    _check(wq.grad, dw, ws, "dq_weight", 100 * 2.0 ** -24)
    assert wk.grad is None
    wq.grad = None
    b = k.clone().requires_grad_()
    qo, ko = norm_rotary(q, b, pos, rot, norm)
    ko[..., 1::2].sum().backward()                                    # only the keys' output is used
    one[..., ::2] = 0
    dx, dw, xs, ws = _gradients(k, one, wk.detach(), pos, rot, norm.eps)
    _check(b.grad, dx, xs, "dk of a slice", BWD)
    _check(wk.grad, dw, ws, "dk_weight", 100 * 2.0 ** -24)
    assert wq.grad is None
    # weights alone; no weights; no keys
    wk.grad = None
    qo, ko = norm_rotary(q, k, pos, rot, norm)
    (qo.sum() + ko.sum()).backward()
    _check(wk.grad, *_gradients(k, torch.ones_like(k), wk.detach(), pos, rot, norm.eps)[1::2], "dk_weight alone", 100 * 2.0 ** -24)
    c = q.clone().requires_grad_()
    qo, none = norm_rotary(c, None, pos, rot, HeadNorm(eps=0.5))
    assert none is None
    qo.backward(torch.ones_like(qo))
    _check(c.grad, *_gradients(q, torch.ones_like(q), None, pos, rot, 0.5)[::2], "dq without weights", BWD)
    # shared heads: a broadcast input's gradient is the sum over its copies, added in bf16 (three roundings)
    d = q[:1].clone().requires_grad_()
    qo, _ = norm_rotary(d.expand(3, 4, 9, 64), None, pos, rot, norm)
    qo.backward(torch.ones_like(qo))
    dx, _, xs, _ = _gradients(q[:1], torch.ones_like(q[:1]), wq.detach(), pos, rot, norm.eps)
    assert ((d.grad.double() - 3 * dx).abs() <= 3 * 2.0 ** -8 * 3 * dx.abs() + 3 * BWD * xs + 1e-5).all()
    # a second derivative is refused
    e = q.float().requires_grad_()
    grad, = torch.autograd.grad(norm_rotary(e, None, pos, rot, HeadNorm())[0].sum(), e, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_strided_in_place_and_layout():
    dev = _cuda()
    from grammar.norm import HeadNorm, norm_rotary_bwd, norm_rotary_fwd
    from grammar.rotary import Rotary
    rot = Rotary(128, rotary_dim=64, device=dev)
    rows = torch.randn((2, 45, 14, 128), device=dev).bfloat16()       # a projection's rows: 8 q, 2 k heads, the rest
    q, k = rows[:, :, :8].transpose(1, 2), rows[:, :, 8:10].transpose(1, 2)
    pos = torch.arange(45, dtype=torch.int32, device=dev)
    norm = HeadNorm(*(1 + 0.2 * torch.randn(128, device=dev) for _ in range(2)))
    keep = rows.clone()
    qo, ko = norm_rotary_fwd(q, k, pos, rot, norm)
    assert torch.equal(rows, keep) and qo.stride(1) < qo.stride(2)    # laid out as q: heads inside tokens
    plain = norm_rotary_fwd(q.contiguous(), k.contiguous(), pos, rot, norm)
    assert torch.equal(qo, plain[0]) and torch.equal(ko, plain[1])
    g = torch.randn((2, 45, 14, 128), device=dev).bfloat16()
    strided = norm_rotary_bwd(q, k, pos, rot, norm, g[:, :, :8].transpose(1, 2), g[:, :, 8:10].transpose(1, 2))
    dense = norm_rotary_bwd(q.contiguous(), k.contiguous(), pos, rot, norm, g[:, :, :8].transpose(1, 2).contiguous(),
                            g[:, :, 8:10].transpose(1, 2).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(strided, dense))
    norm_rotary_fwd(q, k, pos, rot, norm, out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(rows[:, :, 10:], keep[:, :, 10:])              # the neighbours are untouched


def test_rows_that_are_not_finite_stay_their_own():
    """A NaN or an infinity reaches its own row and, as a gradient's sum has it, the weights' gradient; no other row."""
    dev = _cuda()
    from grammar.norm import HeadNorm, norm_rotary_bwd, norm_rotary_fwd
    from grammar.rotary import Rotary
    rot = Rotary(64, device=dev)
    q = torch.randn((1, 3, 20, 64), device=dev)
    norm, pos = HeadNorm(torch.ones(64, device=dev)), torch.arange(20, dtype=torch.int32, device=dev)
    want = norm_rotary_fwd(q, None, pos, rot, norm)[0]
    dq = torch.randn_like(q)
    grad = norm_rotary_bwd(q, None, pos, rot, norm, dq, None, weights=False)[0]
    q[0, 1, 7, 3], q[0, 2, 11, 60] = float("nan"), float("inf")
    got, back = norm_rotary_fwd(q, None, pos, rot, norm)[0], norm_rotary_bwd(q, None, pos, rot, norm, dq, None)[0]
    hit = torch.zeros(1, 3, 20, dtype=torch.bool, device=dev)
    hit[0, 1, 7] = hit[0, 2, 11] = True
    assert torch.equal(got[~hit], want[~hit]) and torch.equal(back[~hit], grad[~hit])
    assert got[0, 1, 7].isnan().all() and got[0, 2, 11].isnan().any() and back[hit].isnan().any(-1).all()


def test_normed_training_attention_gradients():
    """norm_rotary and flash_attention as a training step runs them, against 64 bits."""
    dev = _cuda()
    from grammar.attention import flash_attention
    from grammar.norm import HeadNorm, norm_rotary
    from grammar.rotary import Rotary
    B, H, N, D = 1, 2, 128, 64
    rot = Rotary(D, device=dev)
    pos = torch.arange(N, dtype=torch.int32, device=dev)
    g = torch.Generator("cpu").manual_seed(11)
    q, k, v, do = (torch.randn((B, H, N, D), generator=g).half().to(dev) for _ in range(4))
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dev) for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (q, k, v, wq, wk)]
    qr, kr = norm_rotary(leaves[0], leaves[1], pos, rot, HeadNorm(leaves[3], leaves[4]))
    o = flash_attention(qr, kr, leaves[2], causal=True)
    grads = torch.autograd.grad(o, leaves, do)
    ref = [t.double().clone().requires_grad_() for t in (q, k, v, wq, wk)]
    rq, rk = (_turned(x * w / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6), pos, rot)[0]
              for x, w in ((ref[0], ref[3]), (ref[1], ref[4])))
    s = (rq @ rk.transpose(2, 3).contiguous()) / math.sqrt(D)
    s = s.masked_fill(torch.ones(N, N, dtype=torch.bool, device=dev).triu(1), float("-inf"))
    ro = torch.softmax(s, -1) @ ref[2]
    want = torch.autograd.grad(ro, ref, do.double())
    # fp16 rounds q and k once more than the oracle (2^-11 of scores up to 6 or so), then P, dS and the results: a few
    # 2^-11 of the largest entry; the weights' gradients add B H N such errors of either sign, 2^-11 8 sqrt(256) of an
    # entry's, which are below 1
    for got, w in zip((o, *grads), (ro, *want)):
        unit = max(1.0, float(w.detach().abs().max()))
        assert (got.double() - w).detach().abs().max() <= 8 * 2.0 ** -11 * unit * (16 if w.dim() == 1 else 1)


def test_other_streams_and_graph_replays():
    dev = _cuda()
    from grammar.norm import HeadNorm, norm_rotary, norm_rotary_bwd, norm_rotary_fwd
    from grammar.rotary import Rotary
    rot = Rotary(128, device=dev)
    q, k = (torch.randn((1, h, 77, 128), device=dev).bfloat16() for h in (6, 2))
    pos = torch.arange(77, dtype=torch.int32, device=dev)
    wq, wk = (1 + 0.2 * torch.randn(128, device=dev) for _ in range(2))
    norm = HeadNorm(wq, wk)
    want, back = norm_rotary_fwd(q, k, pos, rot, norm), norm_rotary_bwd(q, k, pos, rot, norm, q, k)
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        out = [torch.zeros_like(t) for t in want]
        side.wait_stream(torch.cuda.current_stream())
        norm_rotary_fwd(q, k, pos, rot, norm, out=out[0], k_out=out[1], stream=stream)
        grads = norm_rotary_bwd(q, k, pos, rot, norm, q, k, stream=stream)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*out, *grads), (*want, *back)))
    leaf, w = q.clone().requires_grad_(), wq.clone().requires_grad_()
    graphs = []
    for _ in range(2):                                                # each with its own workspace
        with torch.cuda.stream(side):
            norm_rotary(leaf, k, pos, rot, HeadNorm(w, wk))
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                qo, ko = norm_rotary(leaf, k, pos, rot, HeadNorm(w, wk))
                dq, dw = torch.autograd.grad(qo, (leaf, w), qo.detach())
        graphs.append((graph, qo, ko, dq, dw))
    torch.cuda.synchronize()
    for i in range(6):
        with torch.no_grad():
            leaf.copy_(torch.randn_like(leaf))
            w.add_(0.01)
            pos.add_(i * 1000)
        graph, qo, ko, dq, dw = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        now = HeadNorm(w.detach(), wk)
        a, b = norm_rotary_fwd(leaf.detach(), k, pos, rot, now)
        assert torch.equal(qo, a) and torch.equal(ko, b)
        x, _, y, _ = norm_rotary_bwd(leaf.detach(), None, pos, rot, now, a, None)
        assert torch.equal(dq, x) and torch.equal(dw, y)


def test_refusals():
    dev = _cuda()
    from grammar import runtime as rt
    from grammar.norm import HeadNorm, norm_rotary, norm_rotary_bwd, norm_rotary_fwd
    from grammar.rotary import Rotary
    rot = Rotary(64, device=dev)
    q, pos = torch.randn((1, 2, 8, 64), device=dev).half(), torch.arange(8, dtype=torch.int32, device=dev)
    w = torch.ones(64, device=dev)
    norm = HeadNorm(w, w)
    for bad in (lambda: norm_rotary_fwd(q.cpu(), None, pos, rot, norm), lambda: norm_rotary_fwd(q, None, pos.long(), rot, norm),
                lambda: norm_rotary_fwd(q, None, pos[:7], rot, norm), lambda: norm_rotary_fwd(q, q.float(), pos, rot, norm),
                lambda: norm_rotary_fwd(q[..., :32], None, pos, rot, norm), lambda: norm_rotary_fwd(None, q, pos, rot, norm),
                lambda: norm_rotary_fwd(q, None, pos, rot, HeadNorm(w[:32])), lambda: norm_rotary_fwd(q, None, pos, rot, HeadNorm(w.cpu())),
                lambda: norm_rotary_fwd(q, None, pos, rot, HeadNorm(w.bfloat16())),
                lambda: norm_rotary_fwd(q, q, pos, rot, HeadNorm(w, w.half())),
                lambda: norm_rotary_fwd(q, None, pos, rot, HeadNorm(torch.ones(128, device=dev)[::2])),
                lambda: norm_rotary_fwd(q, None, pos, rot, norm, out=q[:, :1]), lambda: HeadNorm(w, w, eps=-1.0),
                lambda: HeadNorm(w, w, eps=float("nan")), lambda: norm_rotary_bwd(q, None, pos, rot, norm, q[:, :1], None),
                lambda: norm_rotary_bwd(q, q, pos, rot, norm, q, None), lambda: norm_rotary_bwd(q, None, pos, rot, norm, q.float(), None),
                lambda: norm_rotary_fwd(q.double(), None, pos, rot, norm)):
        with pytest.raises(ValueError):
            bad()
    to = torch.empty_like(q)
    with pytest.raises(ValueError, match="two tensors"):
        norm_rotary_fwd(q, q, pos, rot, norm, out=to, k_out=to)
    rows = torch.randn((1, 8, 6, 64), device=dev).half().transpose(1, 2)
    with pytest.raises(rt.GrError, match="shares memory"):
        norm_rotary_fwd(rows[:, :3], rows[:, 3:5], pos, rot, norm, out=rows[:, 2:5])
    with pytest.raises(rt.GrError, match="aligned"):
        norm_rotary_fwd(q, None, pos, rot, HeadNorm(torch.ones(65, device=dev)[1:]))
    with pytest.raises(rt.GrError, match="multiples of 8"):
        norm_rotary_fwd(torch.randn((1, 2, 8, 68), device=dev).half()[..., :64], None, pos, rot, norm)
    with pytest.raises(NotImplementedError):
        with torch.autograd.forward_ad.dual_level():
            norm_rotary(torch.autograd.forward_ad.make_dual(q.float(), q.float()), None, pos, rot, norm)
    assert norm_rotary_fwd(q[:, :, :0], None, pos[:0], rot, norm)[0].shape == (1, 2, 0, 64)
    none = norm_rotary_bwd(q[:, :, :0], None, pos[:0], rot, norm, q[:, :, :0], None)
    assert none[0].shape == (1, 2, 0, 64) and not none[2].any()
