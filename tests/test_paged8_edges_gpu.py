"""Normed heads and the quantised paged cache at the edges of what their calls promise."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_norm_gpu import _inputs  # noqa: E402
from test_paged_edges_gpu import HINTS  # noqa: E402
from test_paged_gpu import _attention, _cuda  # noqa: E402
from test_paged8_gpu import Setup8, _check, _dequantised  # noqa: E402


@pytest.mark.parametrize("hints", HINTS, ids=lambda h: "-".join(f"{k[4:]}{v}" for k, v in h.items()))
@pytest.mark.parametrize("dtype,D,G,Hkv", [("bf16", 128, 4, 2), ("fp16", 64, 1, 4)])
@pytest.mark.parametrize("width", [None, 2048], ids=["fit", "roomy"])
def test_hints_that_do_not_hold(hints, dtype, D, G, Hkv, width):
    """A packed batch of chunks and single tokens, decode steps over long contexts, drafted tokens and a chunk of its own,
    with hints too small (chunks in tiles of 16 rows) and too large."""
    from grammar.paged import paged_attention
    print(f"[case] hints {hints} {dtype} D{D} width {width}", flush=True)
    for news, lens, ragged in (([1, 0, 150, 1, 7, 301, 1], [40, 99, 150, 700, 7, 900, 0], True),
                               ([1, 1, 1], [20_011, 3, 5000], False), ([6, 6], [2000, 9], False), ([200], [5000], False)):
        s = Setup8(lens, Hkv, 16, D, dtype, seed=D, width=width)
        T, B, Hq = sum(news) + 3 * ragged, len(news), G * Hkv
        q = s.randn(T, Hq, D) if ragged else s.randn(B, Hq, news[0], D)
        starts = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device=s.dev) if ragged else None
        out, lse = torch.full_like(q, 5.0), torch.full((T, Hq) if ragged else (B, news[0], Hq), 7.0, device=s.dev)
        paged_attention(q, s.cache, s.table, s.lens, starts=starts, out=out, lse=lse, **hints)
        for b, n in enumerate(news):
            if n == 0:
                continue
            pick = (lambda x: x[sum(news[:b]):sum(news[:b + 1])]) if ragged else (lambda x: x[b].transpose(0, 1))
            o, ls, size = _attention(s, b, pick(q))
            tol = _check(pick(out), o, size, pick(q), s, b, f"{n} of {lens[b]} keys")
            got, none = pick(lse) if ragged else lse[b], ls == -math.inf
            assert torch.equal(got == -math.inf, none) and ((got.double() - ls).abs() <= tol)[~none].all()
        if ragged:
            assert (out[sum(news):] == 5.0).all() and (lse[sum(news):] == 7.0).all()


@pytest.mark.parametrize("D,hint", [(64, 1), (64, 0), (128, 1), (128, 0)])
def test_overlapping_starts_stay_in_bounds(D, hint):
    """Every second sequence claims all of the batch's rows: more tiles than the grid has. The rows of no other call are
    touched, and every row gets the result that any of them would give."""
    from grammar.paged import paged_attention
    B, rows, W = 512, 16_384, 65_536
    print(f"[case] overlapping starts D{D} hint {hint}", flush=True)
    s = Setup8([16], 2, 16, D, "bf16")
    table = torch.full((1, W), -1, dtype=torch.int32, device=s.dev).expand(B, W)
    lens = torch.full((B,), W * 4, dtype=torch.int32, device=s.dev)
    starts = torch.tensor([0, rows] * (B // 2) + [0], dtype=torch.int32, device=s.dev)
    q = s.randn(rows, 2, D)
    for ws in (None, torch.empty(0, dtype=torch.uint8, device=s.dev)):
        out = torch.full((rows + 64, 2, D), 5.0, dtype=s.dtype, device=s.dev)
        paged_attention(q, s.cache, table, lens, starts=starts, max_new=hint, out=out[32:-32], workspace=ws)
        torch.cuda.synchronize()
        assert not out[32:-32].any() and (out[:32] == 5.0).all() and (out[-32:] == 5.0).all()


@pytest.mark.parametrize("dtype,D,Hkv,width", [("bf16", 128, 24, None), ("fp16", 64, 28, 2048), ("bf16", 64, 40, None)])
def test_part_filled_tiles_in_place(dtype, D, Hkv, width):
    """Results over their own queries, where chunks end in tiles that are done in two passes of 32 rows."""
    from grammar.paged import paged_attention
    news, lens = [129, 388, 160, 289, 191, 64, 40, 5, 193], [140, 388, 500, 300, 191, 64, 700, 5, 260]
    print(f"[case] in place {dtype} D{D} Hkv{Hkv} width {width}", flush=True)
    s = Setup8(lens, Hkv, 16, D, dtype, seed=Hkv, width=width)
    starts = torch.tensor([0] + [sum(news[:b + 1]) for b in range(len(news))], dtype=torch.int32, device=s.dev)
    q = s.randn(sum(news), Hkv, D)
    want = paged_attention(q, s.cache, s.table, s.lens, starts=starts)
    assert paged_attention(q, s.cache, s.table, s.lens, starts=starts, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("pad,off", [(128, 8), (128, 32), (136, 0), (192, 0)])
def test_destinations_off_a_line(pad, off):
    """Normed rows, appended queries and read rows that begin off a 128-byte line: bit for bit the packed ones, and
    nothing behind a row is written."""
    from grammar.norm import HeadNorm, norm_rotary_fwd
    from grammar.paged import paged_append, paged_read
    from grammar.rotary import Rotary
    s = Setup8([700, 900], 8, 16, 128, "bf16", seed=8)
    rot, norm = Rotary(128, device=s.dev), HeadNorm(*(1 + 0.2 * torch.randn(128, device=s.dev) for _ in range(2)))
    print(f"[case] rows of {pad}, {off} off", flush=True)

    def rows(*shape):
        n = math.prod(shape)
        x = torch.full((n * pad + 64,), 5.0, dtype=s.dtype, device=s.dev)
        whole = x[off:off + n * pad].view(*shape, pad)
        return whole[..., :128], lambda: (whole[..., 128:] == 5.0).all() and (x[:off] == 5.0).all() and (x[off + n * pad:] == 5.0).all()
    q, k = s.randn(2, 32, 600, 128), s.randn(2, 8, 600, 128)
    pos = torch.arange(600, dtype=torch.int32, device=s.dev)
    (o, o_kept), (ko, ko_kept) = rows(2, 32, 600), rows(2, 8, 600)
    want = norm_rotary_fwd(q, k, pos, rot, norm)
    norm_rotary_fwd(q, k, pos, rot, norm, out=o, k_out=ko)
    assert torch.equal(o, want[0]) and torch.equal(ko, want[1]) and o_kept() and ko_kept()
    o, o_kept = rows(2, 32, 600)
    want = paged_append(k, k, s.cache, s.table, s.lens, q=q, rotary=rot, norm=norm)
    paged_append(k, k, s.cache, s.table, s.lens, q=q, rotary=rot, norm=norm, out=o)
    assert torch.equal(o, want) and o_kept()
    (ko, ko_kept), (vo, vo_kept) = rows(2, 8, 1000), rows(2, 8, 1000)
    want = paged_read(s.cache, s.table, s.lens, 1000)
    paged_read(s.cache, s.table, s.lens, k_out=ko, v_out=vo)
    assert torch.equal(ko, want[0]) and torch.equal(vo, want[1]) and ko_kept() and vo_kept()


@pytest.mark.parametrize("B,N,Hq,Hk,D,dtype", [(2, 33, 9, 3, 128, "bf16"), (1, 40, 5, 4, 80, "fp16"), (2, 2100, 16, 4, 64, "fp32")])
def test_gradients_in_place(B, N, Hq, Hk, D, dtype):
    """dq and dk over dq_out and dk_out, as the C entry allows: bit for bit those of their own."""
    dev = _cuda()
    from grammar import runtime as rt
    from grammar.norm import norm_rotary_bwd
    from grammar.rotary import check_positions, head_strides
    print(f"[case] in place B{B} N{N} H{Hq}/{Hk} D{D} {dtype}", flush=True)
    g, rot, norm, q, k, pos = _inputs(B, N, Hq, Hk, D, D // 32 * 16, None, False, dtype, "fp32", dev)
    dq, dk = (torch.randn(t.shape, generator=g).to(t.dtype).to(dev) for t in (q, k))
    want = norm_rotary_bwd(q, k, pos, rot, norm, dq, dk)
    L, code, spec = rt.lib(), rt.dtype_code(q.dtype), norm.spec(D, q.dtype, rot.index, "test")
    need = L.gr_norm_rotary_bwd_workspace(Hq, Hk, D, B, N)
    ws, wq, wk = torch.empty(need, dtype=torch.uint8, device=dev), torch.empty(D, device=dev), torch.empty(D, device=dev)

    def side(x, d):
        st = head_strides(x, "x", "test")
        return x.data_ptr(), d.data_ptr(), d.data_ptr(), x.shape[1], st, st, st
    rt.launch(L.gr_norm_rotary_bwd, (rot.ref, ctypes.addressof(spec)) + side(q, dq) + side(k, dk) +
              (code, B, N, pos.data_ptr(), check_positions(pos, rot, (B, N), "test"), wq.data_ptr(), wk.data_ptr(), ws.data_ptr(), need),
              q, None, "gr_norm_rotary_bwd")
    for a, b in zip((dq, dk, wq, wk), want):
        assert torch.equal(a, b)


def test_one_tensor_for_queries_and_keys_and_one_weight_for_both():
    """The gradients of a tensor that is both add up, as torch has it."""
    dev = _cuda()
    from grammar.norm import HeadNorm, norm_rotary, norm_rotary_bwd
    from grammar.rotary import Rotary
    rot, pos = Rotary(64, device=dev), torch.arange(30, dtype=torch.int32, device=dev)
    x = torch.randn((2, 5, 30, 64), device=dev).requires_grad_()
    w = (1 + 0.2 * torch.randn(64, device=dev)).requires_grad_()
    a, b = torch.randn_like(x), torch.randn_like(x)
    q, k = norm_rotary(x, x, pos, rot, HeadNorm(w, w))
    assert torch.equal(q, k) and q.data_ptr() != k.data_ptr()
    dx, dw = torch.autograd.grad((q, k), (x, w), (a, b))
    y, v = x.detach(), w.detach()
    dq, dk, wq, wk = norm_rotary_bwd(y, y, pos, rot, HeadNorm(v, v), a, b)
    assert torch.equal(dx, dq + dk) and torch.equal(dw, wq + wk)


@pytest.mark.parametrize("D,S", [(64, 1 << 20), (128, 1 << 16)])
def test_one_large_page(D, S):
    """A page holds a whole sequence, its scales side by side."""
    from grammar.paged import QuantizedPagedCache, paged_append, paged_attention, paged_read
    dev = _cuda()
    cache = QuantizedPagedCache.empty(2, 1, S, D, torch.float16, device=dev)
    for t in (cache.k, cache.v, cache.scales):
        t.view(torch.uint8).fill_(0x7f)                               # NaN, and scales of 1
    s = Setup8([5000], 1, 16, D, "fp16", seed=1)
    table = torch.tensor([[1]], dtype=torch.int32, device=dev)
    k, v, q = s.randn(1, 1, 5000, D), s.randn(1, 1, 5000, D), s.randn(1, 4, 100, D)
    for c, t in ((cache, table), (s.cache, s.table)):
        paged_append(k, v, c, t, s.lens)
    for a, b in zip(paged_read(cache, table, s.lens, 5100), paged_read(s.cache, s.table, s.lens, 5100)):
        assert torch.equal(a, b) and not a[:, :, 5000:].any()
    none = torch.empty(0, dtype=torch.uint8, device=dev)              # (a workgroup a tile: shares go by the table's size)
    for n in (1, 7, 100):
        args = dict(max_len=5000, workspace=none)
        assert torch.equal(paged_attention(q[:, :, -n:], cache, table, s.lens, **args), paged_attention(q[:, :, -n:], s.cache, s.table, s.lens, **args))
        o = paged_attention(q[:, :, -n:], cache, table, s.lens)        # shared out by 2^20 keys
        sc = s.cache.scales
        s.k, s.v = (_dequantised(t, sc[:, :, j].contiguous()).to(s.dtype) for j, t in enumerate((s.cache.k, s.cache.v)))
        ref, _, size = _attention(s, 0, q[0, :, -n:].transpose(0, 1))
        _check(o[0].transpose(0, 1), ref, size, q[0, :, -n:].transpose(0, 1), s, 0, f"{n} tokens")
