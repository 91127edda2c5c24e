"""The quantised paged cache: appending (gr_paged_append_with), attention over it
(gr_paged_attn_scaled) and reading back (gr_paged_read) against the definitions in
64 bits, at the lengths, masks, pages, values and layouts where they can go wrong."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_norm_gpu import FWD, _normed, _size  # noqa: E402
from test_paged_gpu import APPENDS, LENS, Setup, _attention, _cuda, _rotated  # noqa: E402

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _scale_of(top):
    """E8M0 bytes for rows whose largest magnitude is `top` (64 bits): the least k from -127 on with top <= 448 2^k."""
    m, e = torch.frexp(top)
    return (torch.where(top > 0, e - 9 + (m > 0.875), torch.full_like(e, -127)).clamp(min=-127) + 127).to(torch.uint8)


def _clamped(x, dtype):
    """x within the largest numbers of four significant bits in the type."""
    most = 61440.0 if dtype == torch.float16 else 15 * 2.0 ** 124
    return x.clamp(-most, most)


def _quantised(x, dtype):
    """(e4m3, E8M0) of finite rows x, by the definition in 64 bits."""
    x = _clamped(x.double(), dtype)
    sb = _scale_of(x.abs().amax(-1))
    # (a 64-bit number to e4m3 by way of fp32: at most 11 significant bits come in, so nothing rounds twice)
    return torch.ldexp(x, 127 - sb.int().unsqueeze(-1)).float().to(E4M3), sb.view(E8M0)


def _dequantised(v, sb):
    s = torch.exp2(sb.view(torch.uint8).double() - 127)
    return v.double() * torch.where(sb.view(torch.uint8) == 255, float("nan"), s).unsqueeze(-1)


class Setup8(Setup):
    """A Setup whose cache is quantised; k and v are what it stands for."""

    def __init__(self, *args, spread=1.0, **kw):
        from grammar.paged import QuantizedPagedCache
        super().__init__(*args, **kw)
        for t in (self.k, self.v):
            t.mul_(torch.exp2(spread * torch.randn(t.shape[:3], generator=self.g)).to(self.dev).unsqueeze(-1).to(self.dtype))
        self.put()

    def put(self):
        """The cache of k and v as they are; they become what it stands for."""
        from grammar.paged import QuantizedPagedCache
        odd = {}
        for n in "kv":
            x = getattr(self, n)
            odd[n] = ~x.isfinite()
        (kq, ks), (vq, vs) = (_quantised(torch.where(odd[n], torch.zeros_like(getattr(self, n)), getattr(self, n)), self.dtype) for n in "kv")
        scales = torch.stack((ks.view(torch.uint8), vs.view(torch.uint8)), 2).contiguous()
        for i, (n, q) in enumerate((("k", kq), ("v", vq))):
            hit = odd[n].any(-1)
            q.view(torch.uint8)[hit] = 0x7f
            scales[:, :, i][hit] = 255
        self.scales = scales.view(E8M0)
        self.kq, self.vq = kq, vq
        self.cache = QuantizedPagedCache(kq, vq, self.scales, self.dtype)
        self.k, self.v = (_dequantised(q, scales[:, :, i].contiguous().view(E8M0)).to(self.dtype) for i, q in enumerate((kq, vq)))
        return self


def _check(got, want, size, q, s, b, what, scale=None):
    """The result [n, Hq, D] of sequence b's tokens q against `want`; returns what the log-sum-exp may be off.

    Rows' weights p_j are taken relative to a base that a key has reached, so that their sum l is 1 at least.
     scores: D products added in some order, 2^-24 of their sizes' sum A each; scaled and shifted by the base,
             2^-24 of both a few times; 2^x to 2^-23. Each p is off by e = 2^-24 ((D + 8) A + 8) of itself.
     P:      rounds to the type, u = half a step of itself; in fp16 below 2^-14 by 2^-25, less by the 2^shift that P
             carries over more than 2,048 keys: `sub` for each key.
     result: sum p v / l, both with e, u and sub, and one rounding more (fp16 below 2^-14: 2^-25)."""
    k, v = s.keys(b, s.k)[0], s.keys(b, s.v)[0]
    n, Hq, D = q.shape
    G, m = Hq // k.shape[0], k.shape[1]
    u = torch.finfo(got.dtype).eps / 2
    if m == 0:
        assert not got.any(), what
        return torch.zeros(n, Hq, dtype=torch.float64, device=q.device)
    ka, va = (t.nan_to_num(0, 0, 0).abs().repeat_interleave(G, 0) for t in (k, v))
    A = torch.matmul(q.double().abs().transpose(0, 1), ka.transpose(1, 2).contiguous()).amax(-1).T * (scale or 1 / math.sqrt(D))
    e = (2.0 ** -24 * ((D + 8) * A + 8)).unsqueeze(-1)                # [n, Hq, 1]
    sub = 2.0 ** -(25 + max(0, (m - 1).bit_length() - 11)) if got.dtype == torch.float16 else 0.0
    o = want.nan_to_num(0, 0, 0).abs()
    tol = (u + e) * (size + o) + sub * (va.sum(1) + m * o) + u * o
    tol = tol * 1.01 + (2.0 ** -24 if got.dtype == torch.float16 else 2.0 ** -120)
    bad = ~((got.double() - want).abs() <= tol) & want.isfinite()
    bad |= want.isnan() != got.isnan()
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() - tol).max())}"
    # m and l: e and the roundings of l's terms, one of the base in natural units and of the logarithm
    return (u + e[..., 0] + sub * m) * 1.01 + 2.0 ** -22 * (A + 8)


def _run(s, news, Hq, causal=True, ragged=False, pad=0, hints=True, strided=False, workspace=None):
    """paged_attention of `news` new tokens a sequence, checked row by row; returns the result."""
    from grammar.paged import paged_attention
    B, D = len(s.lens_host), s.D
    T = sum(news) + pad
    if ragged:
        q = s.randn(T, Hq + 2, D)[:, 1:-1] if strided else s.randn(T, Hq, D)
        starts = torch.tensor([0] + [sum(news[:b + 1]) for b in range(B)], dtype=torch.int32, device=s.dev)
        lse = torch.full((T, Hq), 7.0, device=s.dev)
        out = torch.full((T, Hq, D), 5.0, device=s.dev, dtype=s.dtype)
    else:
        n = news[0]
        assert set(news) == {n}
        q = s.randn(B, n, Hq + 2, D)[:, :, 1:-1].transpose(1, 2) if strided else s.randn(B, Hq, n, D)
        starts, lse = None, torch.full((B, n, Hq), 7.0, device=s.dev)
        out = torch.full(q.shape, 5.0, device=s.dev, dtype=s.dtype)
    more = dict(max_new=max(news), max_len=max(1, max(s.lens_host))) if hints else {}
    got = paged_attention(q, s.cache, s.table, s.lens, starts=starts, causal=causal, out=out, lse=lse, workspace=workspace,
                          **more)
    torch.cuda.synchronize()
    assert got is out
    row = 0
    for b, n in enumerate(news):
        qb, ob = (x[row:row + n] if ragged else x[b].transpose(0, 1) for x in (q, out))
        lb = lse[row:row + n] if ragged else lse[b]
        row += n
        if n == 0:
            continue
        o, ls, size = _attention(s, b, qb, causal)
        tol = _check(ob, o, size, qb, s, b, f"sequence {b}: {n} tokens, {s.lens_host[b]} keys")
        if o.isfinite().all():
            none = ls == -math.inf
            assert torch.equal(lb == -math.inf, none), f"lse of sequence {b}"
            assert ((lb.double() - ls).abs() <= tol)[~none].all(), f"lse of sequence {b}"
    if ragged:
        assert (out[row:] == 5.0).all() and (lse[row:] == 7.0).all()      # rows behind the last sequence
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_every_number_and_scale_reads_back_exactly(dtype):
    """All 256 bytes under all 256 scales, as far as the tokens' type holds what they stand for."""
    from grammar.paged import QuantizedPagedCache, paged_read
    dev, dt = _cuda(), {"fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    k = torch.arange(256, dtype=torch.uint8, device=dev).view(1, 4, 1, 64).expand(16, 4, 16, 64).contiguous()
    sb = torch.arange(256, dtype=torch.uint8, device=dev).view(16, 1, 1, 16).expand(16, 4, 2, 16).contiguous()
    cache = QuantizedPagedCache(k.view(E4M3), k.flip(3).contiguous().view(E4M3), sb.view(E8M0), dt)
    table = torch.arange(16, dtype=torch.int32, device=dev).view(1, 16)
    got = paged_read(cache, table, torch.tensor([256], dtype=torch.int32, device=dev), 256)
    for x, q in zip(got, (cache.k, cache.v)):
        want = _dequantised(q, sb[:, :, 0].contiguous().view(E8M0)).transpose(1, 2).reshape(256, 4, 64).transpose(0, 1)[None]
        held = want.abs() <= torch.finfo(dt).max                     # (NaN: no)
        assert torch.equal(x[held].double(), want[held].to(dt).double())
        assert torch.equal(x.isnan(), want.isnan())


# ---- attention: what holds over the 16-bit cache holds over what this one stands for ----------

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,Hkv,S", [(1, 3, 16), (4, 2, 16), (7, 1, 64), (16, 1, 32), (40, 1, 16), (70, 1, 128)])
def test_single_tokens(dtype, D, G, Hkv, S):
    print(f"[case] decode {dtype} D{D} G{G} Hkv{Hkv} S{S}", flush=True)
    s = Setup8(LENS, Hkv, S, D, dtype, seed=G)
    _run(s, [1] * len(LENS), G * Hkv)
    _run(s, [1] * len(LENS), G * Hkv, ragged=True, pad=3, hints=False, strided=True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G,Hkv", [(2, 1, 2), (5, 7, 1), (13, 5, 2), (33, 1, 2), (64, 2, 1), (100, 3, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_few_tokens(dtype, D, n, G, Hkv, causal):
    lens = [n, n + 1, n + 16, max(0, n - 3), 0, 1, 3 * n + 70, 513]
    print(f"[case] few {dtype} D{D} n{n} G{G} causal={causal}", flush=True)
    s = Setup8(lens, Hkv, 16, D, dtype, seed=n)
    _run(s, [n] * len(lens), G * Hkv, causal=causal, strided=True)


@pytest.mark.parametrize("dtype,D,G,Hkv,S", [("bf16", 128, 4, 2, 16), ("fp16", 64, 1, 4, 32), ("bf16", 64, 6, 1, 128),
                                             ("fp16", 128, 3, 2, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_mixed_batches(dtype, D, G, Hkv, S, causal):
    news = [1, 0, 150, 1, 7, 0, 1, 301, 1, 0]
    lens = [40, 99, 150, 700, 7, 0, 1, 900, 0, 5]
    print(f"[case] mixed {dtype} D{D} G{G} Hkv{Hkv} S{S} causal={causal}", flush=True)
    s = Setup8(lens, Hkv, S, D, dtype, seed=D + G)
    _run(s, news, G * Hkv, causal=causal, ragged=True, pad=9)
    _run(s, news, G * Hkv, causal=causal, ragged=True, hints=False)


def test_more_sequences_than_a_wave_has_lanes():
    rng = random.Random(3)
    news = [rng.choice((0, 1, 1, 1, 3, 40)) for _ in range(150)]
    lens = [n + rng.choice((0, 0, 1, 30, 200)) for n in news]
    _run(Setup8(lens, 2, 16, 64, "bf16", seed=4), news, 6, ragged=True, pad=2)


def _needs_workspace(s, rows, Hq, starts=None):
    import ctypes
    from grammar import runtime as rt
    batch = rt.PagedBatch(s.table.data_ptr(), s.width, s.lens.data_ptr(), starts, len(s.lens_host), rows, s.width, 0, 0)
    return int(rt.lib().gr_paged_attn_scaled_workspace(s.cache.ref, s.cache.scales_ref, ctypes.addressof(batch), Hq))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G,Hkv", [(1, 4, 2), (1, 1, 3), (5, 7, 1), (3, 20, 1), (50, 4, 1)])
def test_shared_work_of_ragged_lengths(dtype, D, n, G, Hkv):
    lens = [m + n - 1 for m in LENS] + [0, 3000, 64, 128, 5000, n]
    s = Setup8(lens, Hkv, 16, D, dtype, seed=n, width=1024)
    print(f"[case] shared {dtype} D{D} n{n} G{G} Hkv{Hkv}", flush=True)
    assert _needs_workspace(s, n, G * Hkv) > 0
    _run(s, [n] * len(lens), G * Hkv, hints=False, strided=True)


@pytest.mark.parametrize("dtype,D,G,Hkv", [("bf16", 128, 4, 2), ("fp16", 64, 1, 2)])
def test_shared_mixed_batches(dtype, D, G, Hkv):
    news = [1, 0, 150, 1, 7, 0, 1, 301, 1, 0] + [1] * 70
    lens = [40, 99, 150, 4000, 7, 0, 1, 900, 0, 5] + [3 * i for i in range(70)]
    s = Setup8(lens, Hkv, 16, D, dtype, seed=D, width=2048)
    print(f"[case] shared mixed {dtype} D{D} G{G}", flush=True)
    assert _needs_workspace(s, sum(news) + 5, G * Hkv, s.lens.data_ptr()) > 0
    for causal in (True, False):
        _run(s, news, G * Hkv, causal=causal, ragged=True, pad=5, hints=False)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("G,Hkv", [(8, 16), (4, 8), (2, 8)], ids=["many", "few", "small"])
def test_mixed_batches_of_a_workgroup_a_tile(dtype, D, G, Hkv):
    """Tiles of 128 rows in grids that fill the GPU and that do not, and of 32 rows."""
    news = [1, 130, 0, 33, 300, 1, 16] + [1, 0, 2] * 25 + [34]
    lens = [260, 131, 9, 33, 449, 0, 80] + [5 * i for i in range(75)] + [70]
    s = Setup8(lens, Hkv, 32, D, dtype, seed=G)
    print(f"[case] tiles {dtype} D{D} G{G} Hkv{Hkv}", flush=True)
    assert _needs_workspace(s, sum(news) + 3, G * Hkv, s.lens.data_ptr()) == 0
    for causal in (True, False):
        _run(s, news, G * Hkv, causal=causal, ragged=True, pad=3, hints=False)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("news,lens,G,Hkv", [([2049] + [1] * 8, [2300, 700, 5, 900, 0, 33, 64, 65, 1500], 4, 8),
                                             ([513, 0, 700], [513, 9, 1900], 8, 9), ([1100] * 3, [1100, 1500, 1900], 4, 5)])
def test_long_chunks(dtype, D, news, lens, G, Hkv):
    """Tiles of 128 rows, in packed and uniform batches, with room in the grid for tiles that the lengths do not make."""
    print(f"[case] chunks {dtype} D{D} {news} G{G} Hkv{Hkv}", flush=True)
    s = Setup8(lens, Hkv, 64, D, dtype, seed=D)
    uniform = len(set(news)) == 1
    for causal in (True, False):
        _run(s, news, G * Hkv, causal=causal, ragged=not uniform, pad=0 if uniform else 200, hints=causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
def test_long_contexts_share_their_keys_out(D, n):
    from grammar.paged import paged_attention
    s = Setup8([20_011, 3, 5000], 2, 32, D, "bf16", seed=D)
    print(f"[case] long D{D} n{n}", flush=True)
    _run(s, [n] * 3, 8)
    q = s.randn(3, 8, n, D)
    need = _needs_workspace(s, n, 8)
    assert need > 0
    for size in (need, need // 2, need // 5, need // 100, 16, 0):
        ws = torch.empty(size, dtype=torch.uint8, device=s.dev)
        a, b = (paged_attention(q, s.cache, s.table, s.lens, workspace=ws) for _ in range(2))
        assert torch.equal(a, b)
        for i in range(3):
            o, _, sz = _attention(s, i, q[i].transpose(0, 1))
            _check(a[i].transpose(0, 1), o, sz, q[i].transpose(0, 1), s, i, f"workspace {size}, sequence {i}")


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("fp16", 128)])
@pytest.mark.parametrize("n,G,Hkv", [(1, 4, 2), (9, 4, 2), (70, 2, 2), (90, 8, 24), (90, 4, 12)])
@pytest.mark.parametrize("width", [None, 2048], ids=["tile", "shared"])
def test_hidden_entries_may_hold_anything(dtype, D, n, G, Hkv, width):
    """Stale slots and pages of other sequences hold NaN, bytes and scales; a row that only later tokens see is NaN, and
    so are they, but no earlier row. Pages that do not exist at a sequence's start and middle."""
    lens = [n, n + 7, n + 100, 200 + n]
    s = Setup8(lens, Hkv, 16, D, dtype, seed=n, width=width)
    nan = float("nan")
    live = torch.zeros(s.k.shape[0], s.S, dtype=torch.bool)
    for b, m in enumerate(lens):
        for j in range(m):
            live[int(s.table[b, j // s.S]), j % s.S] = True
    dead = (~live).to(s.dev)[:, None, :, None]
    s.k.masked_fill_(dead, nan)
    s.v.masked_fill_(dead, nan)
    s.put()
    s.table[2, 0], s.table[3, 5], s.table[3, 9] = s.k.shape[0], -9, 2 ** 31 - 1
    print(f"[case] hidden {dtype} D{D} n{n} G{G} width {width}", flush=True)
    assert _run(s, [n] * 4, Hkv * G, hints=False).isfinite().all()
    if n == 1:
        return
    # the last token's entries: a NaN key in head 0, a NaN value in head 1
    for b, m in enumerate(lens[:2]):
        page, slot = int(s.table[b, (m - 1) // s.S]), (m - 1) % s.S
        s.k[page, 0, slot, 3] = nan
        s.v[page, 1, slot, 5] = nan
    s.put()
    out = _run(s, [n] * 4, Hkv * G, hints=False)
    assert out[:, :, :-1].isfinite().all()                      # earlier rows
    assert out[:2, :2 * G, -1].isnan().all() and out[:2, 2 * G:].isfinite().all()


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("fp16", 128)])
@pytest.mark.parametrize("Hkv,width", [(24, None), (28, 2048), (40, None)], ids=["two groups", "shared", "tile"])
@pytest.mark.parametrize("causal", [True, False])
def test_part_filled_tiles_of_chunks(dtype, D, Hkv, width, causal):
    """Chunks that end in a tile of 1, 4, 32, 33, 63, 64 and 65 of 128 rows, among sequences of as few; stale slots are
    NaN, a page does not exist, and the last token of two sequences is NaN, which only rows that see it show."""
    news = [129, 388, 160, 289, 191, 64, 40, 5, 193]
    lens = [140, 388, 500, 300, 150, 64, 700, 5, 260]
    print(f"[case] part-filled {dtype} D{D} Hkv{Hkv} causal={causal}", flush=True)
    s = Setup8(lens, Hkv, 16, D, dtype, seed=Hkv, width=width)
    live = torch.zeros(s.k.shape[0], s.S, dtype=torch.bool)
    for b, m in enumerate(lens):
        for j in range(m):
            live[int(s.table[b, j // s.S]), j % s.S] = True
    dead = (~live).to(s.dev)[:, None, :, None]
    s.k.masked_fill_(dead, float("nan"))
    s.v.masked_fill_(dead, float("nan"))
    if causal:
        for b in (0, 3):
            page, slot = int(s.table[b, (lens[b] - 1) // s.S]), (lens[b] - 1) % s.S
            s.k[page, 0, slot, 3] = s.v[page, 1, slot, 5] = float("nan")
    s.put()
    s.table[6, 7], s.table[2, 0] = -1, s.k.shape[0]
    out = _run(s, news, Hkv, causal=causal, ragged=True, pad=3)
    bad = out.isnan().any(-1).any(-1).nonzero().flatten().tolist()
    last = [sum(news[:b + 1]) - 1 for b in (0, 3)]
    assert bad == (last if causal else [])


@pytest.mark.parametrize("width", [None, 2048], ids=["tile", "shared"])
def test_pages_that_do_not_exist(width):
    from grammar.paged import paged_attention
    s = Setup8([100, 100, 64], 2, 16, 64, "bf16", seed=1, width=width)
    s.table[0, 2], s.table[0, 6], s.table[1, 0] = -1, s.k.shape[0], 2 ** 31 - 1
    s.table[2, :4] = -7
    for n in (1, 20):
        out = _run(s, [n] * 3, 4, hints=False)
        assert not out[2].any()
    for m in (50_000, -5):                                      # more keys than the table holds; fewer than none
        s.lens_host[1] = m
        s.lens.copy_(torch.tensor(s.lens_host, dtype=torch.int32))
        out = _run(s, [3] * 3, 4, hints=False)
        assert m > 0 or not out[1].any()
    q = s.randn(6, 4, 64)
    out = torch.full_like(q, 5.0)
    for starts in ([0, 3, 2, 9], [-4, -1, 7, 100], [6, 6, 6, 6]):
        paged_attention(q, s.cache, s.table, s.lens, starts=torch.tensor(starts, dtype=torch.int32, device=s.dev), out=out)
        torch.cuda.synchronize()
        assert (out[3:] == 5.0).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("w", [23.4, 25.05])
@pytest.mark.parametrize("n,G,D,alone", [(1, 4, 64, False), (1, 4, 128, True), (200, 2, 128, False), (4100, 8, 64, True)])
def test_many_small_weights_add_up(dtype, w, n, G, D, alone):
    """One key of weight 1 and value 1, then N of about 2^-w and value -1 (as over the 16-bit cache)."""
    from grammar.paged import paged_attention
    N = 50_001
    s = Setup8([N], 1, 64, D, dtype)
    s.k.zero_()
    s.k[..., 0] = -w * math.log(2)
    s.v.fill_(-1.0)
    first = int(s.table[0, 0])
    s.k[first, 0, 0] = 0
    s.v[first, 0, 0] = 1
    s.put()
    x = float(s.k[first, 0, 1, 0])                               # the score as it is stored
    print(f"[case] small weights {dtype} w {w} ({x}) n{n} G{G} D{D} alone={alone}", flush=True)
    q = torch.zeros(1, G, n, D, dtype=s.dtype, device=s.dev)
    q[..., 0] = 1
    lse = torch.empty(1, n, G, device=s.dev)
    got = paged_attention(q, s.cache, s.table, s.lens, scale=1.0, lse=lse,
                          workspace=torch.empty(0, dtype=torch.uint8, device=s.dev) if alone else None)
    m = (N - n + torch.arange(n, dtype=torch.float64, device=s.dev)) * math.exp(x)
    want = ((1 - m) / (1 + m))[None, None, :, None]
    # p, sums and the result as over the 16-bit cache
    u = torch.finfo(s.dtype).eps / 2
    sums = N / 4 * 2.0 ** -24
    off = float(m.max()) * (u + 40 * 2.0 ** -24 + 2.0 ** -22) + (2.0 ** -14 if dtype == "fp16" else 0)
    assert ((got.double() - want).abs() <= 2 * off + sums + u * want.abs()).all(), float((got.double() - want).abs().max())
    assert ((lse.double() - torch.log1p(m)[None, :, None]).abs() <= off + sums + 2.0 ** -22).all()


def test_rows_of_very_different_scales():
    """Keys and values whose scales differ by 2^40 and more, and numbers near the ends of bf16's range."""
    s = Setup8([300, 77], 2, 16, 64, "bf16", seed=3)
    e = torch.randint(-60, 20, s.v.shape[:3], generator=s.g).to(s.dev).double()
    s.v.copy_((s.v.double() * torch.exp2(e).unsqueeze(-1)).to(s.dtype))
    s.k.mul_(torch.exp2(-torch.rand(s.k.shape[:3], generator=s.g).to(s.dev) * 30).unsqueeze(-1).to(s.dtype))
    page, slot = int(s.table[0, 3]), 5
    s.v[page, 0, slot, :4] = torch.tensor([1e30, -1e30, 1e-38, 0.0], dtype=s.dtype)
    s.put()
    for n in (1, 9, 70):
        _run(s, [n] * 2, 8, hints=False)


def test_cache_layouts_and_table_strides():
    """Pages stored [pages, page_size, heads, D], keys and values in one tensor, scales of their own layout, and a table
    that is a slice."""
    from grammar.paged import QuantizedPagedCache, paged_append, paged_attention, paged_read
    s = Setup8([77, 130, 5], 3, 16, 128, "bf16", seed=9)
    both = torch.stack((s.kq.view(torch.uint8).transpose(1, 2), s.vq.view(torch.uint8).transpose(1, 2)), 2).contiguous().view(E4M3)
    sc = s.scales.view(torch.uint8).permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3).view(E8M0)   # [kind][head][page]
    cache = QuantizedPagedCache(both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), sc, s.dtype)
    table = torch.full((3, 40), 10 ** 6, dtype=torch.int32, device=s.dev)
    table[:, 5:5 + s.width] = s.table
    table = table[:, 5:5 + s.width]
    for n in (1, 4, 60):
        q, k, v = s.randn(3, 6, n, 128), s.randn(3, 3, n, 128), s.randn(3, 3, n, 128)
        for c, t in ((s.cache, s.table), (cache, table)):
            paged_append(k, v, c, t, s.lens)
        assert torch.equal(paged_attention(q, cache, table, s.lens), paged_attention(q, s.cache, s.table, s.lens))
    for a, b in zip(paged_read(cache, table, s.lens, 140), paged_read(s.cache, s.table, s.lens, 140)):
        assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Pages whose bytes, and scales, lie beyond 2^32 of the cache's start."""
    from grammar.paged import QuantizedPagedCache, paged_append, paged_attention, paged_read
    dev = _cuda()
    P, H, S, D = 140_000, 4, 64, 128                             # 4.6e9 bytes each
    cache = QuantizedPagedCache.empty(P, H, S, D, torch.bfloat16, device=dev)
    table = torch.tensor([[P - 1, 0, P - 3, 131_073]], dtype=torch.int32, device=dev)
    g = torch.Generator("cpu").manual_seed(1)
    k, v = (torch.randn((1, H, 250, D), generator=g).bfloat16().to(dev) for _ in range(2))
    lens = torch.tensor([250], dtype=torch.int32, device=dev)
    paged_append(k, v, cache, table, lens)
    s = Setup8([250], H, S, D, "bf16")
    paged_append(k, v, s.cache, s.table, s.lens)
    for a, b, x in zip(paged_read(cache, table, lens, 250), paged_read(s.cache, s.table, s.lens, 250), (k, v)):
        assert torch.equal(a, b) and torch.equal(a.double(), _dequantised(*_quantised(x, torch.bfloat16)))
    q = torch.randn((1, 8, 250, D), generator=g).bfloat16().to(dev)
    for n in (1, 20, 250):
        assert torch.equal(paged_attention(q[:, :, -n:], cache, table, lens), paged_attention(q[:, :, -n:], s.cache, s.table, s.lens))


# ---- appending -------------------------------------------------------------------

def _check_rows(q, sb, want, size, coef, dtype, what):
    """Stored rows (e4m3, E8M0) of values that fp32 has as `want` off by coef * size: the scale is that of some largest
    magnitude within that, the numbers are the nearest ones to some value within it."""
    slack = coef * size
    want = _clamped(want, dtype)
    top = want.abs().amax(-1)
    off = slack.amax(-1)
    sb = sb.view(torch.uint8)
    lo, hi = _scale_of((top - off).clamp(min=0)), _scale_of(top + off)
    assert ((sb >= lo) & (sb <= hi)).all(), what
    # e4m3 under the scale: half a step is 2^(e - 4) 2^k for magnitudes from 2^e to 2^(e + 1), 2^-10 2^k below 2^-6
    unit = torch.exp2(sb.double() - 127).unsqueeze(-1)
    z = want.abs() + slack
    e = torch.floor(torch.log2((z / unit).clamp(min=2.0 ** -6)))
    tol = torch.exp2(e - 4) * unit * (1 + 1e-9) + slack
    got = q.double() * unit
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off"


@pytest.mark.parametrize("news,lens,Hq,Hkv,D,S,rd,sections,inter,dtype,ragged", APPENDS)
@pytest.mark.parametrize("norm,q8", [("same", True), ("fp32", False), (None, True)])
def test_append(news, lens, Hq, Hkv, D, S, rd, sections, inter, dtype, ragged, norm, q8):
    from grammar.norm import HeadNorm
    from grammar.paged import PagedCache, paged_append
    from grammar.rotary import Rotary
    print(f"[case] append {news} D{D} S{S} {sections} {dtype} norm={norm} q8={q8}", flush=True)
    s = (Setup8 if q8 else Setup)(lens, Hkv, S, D, dtype, seed=len(news))
    rot = Rotary(D, rotary_dim=rd, sections=sections, interleaved=inter, device=s.dev)
    hn = None
    if norm:
        hn = HeadNorm(*((1 + 0.3 * torch.randn(D, generator=s.g)).to(torch.float32 if norm == "fp32" else s.dtype).to(s.dev)
                        for _ in range(2)))
    pad = 4 if ragged else 0
    T, B = sum(news) + pad, len(news)
    rows = s.randn(T, Hq + 2 * Hkv, D)                            # a projection's rows: q, k, v side by side
    where = rows if ragged else rows.view(B, news[0], Hq + 2 * Hkv, D).transpose(1, 2)
    q, k, v = where.split([Hq, Hkv, Hkv], 1)
    lead = (rot.naxes,) if rot.naxes > 1 else ()
    pos = torch.randint(0, 5000, lead + (T,), generator=s.g, dtype=torch.int32).to(s.dev) if sections else None
    given = None if pos is None else pos if ragged else pos.view(lead + (B, news[0]))
    starts = torch.tensor([0] + [sum(news[:b + 1]) for b in range(B)], dtype=torch.int32, device=s.dev) if ragged else None
    held = [s.cache.k, s.cache.v] + ([s.cache.scales] if q8 else [])
    before = [t.view(torch.uint8).clone() if q8 else t.clone() for t in held]
    out = torch.full_like(q, 5.0)
    got = paged_append(k, v, s.cache, s.table, s.lens, starts=starts, q=q, rotary=rot, norm=hn, out=out, positions=given)
    torch.cuda.synchronize()
    assert got is out
    written = torch.zeros(s.k.shape[0], S, dtype=torch.bool, device=s.dev)
    coef = FWD if norm else 4e-7
    at = 0
    for b, n in enumerate(news):
        place = torch.arange(lens[b] - n, lens[b], device=s.dev)
        p = pos[..., at:at + n] if pos is not None else place.expand(lead + (n,))
        pick = (lambda x: x[at:at + n]) if ragged else (lambda x: x[b].transpose(0, 1))

        def turned(x, w):
            y, size = _rotated(_normed(x, w, hn.eps)[0] if hn else x, p, rot)
            return y, _size(y, size)
        if n:
            y, size = turned(pick(q), hn and hn.q_weight)
            tol = torch.finfo(s.dtype).eps / 2 * y.abs() * 1.001 + coef * size + 2.0 ** -25
            assert ((pick(out).double() - y).abs() <= tol).all(), f"q of {b}"
        keep = place >= 0
        page, slot = s.table[b].long()[place[keep] // S], place[keep] % S
        if keep.any():
            y, size = turned(pick(k), hn and hn.k_weight)
            y, size, x = y[keep], size[keep], pick(v)[keep]
            if q8:
                kq, vq, sc = (t.view(torch.uint8) for t in held)
                _check_rows(kq[page, :, slot].view(E4M3), sc[page, :, 0, slot], y, size, coef, s.dtype, f"k of {b}")
                want, scale = _quantised(x, s.dtype)
                assert torch.equal(sc[page, :, 1, slot], scale.view(torch.uint8))
                assert torch.equal(vq[page, :, slot].view(E4M3).float(), want.float())
            else:
                tol = torch.finfo(s.dtype).eps / 2 * y.abs() * 1.001 + coef * size + 2.0 ** -25
                assert ((s.k[page, :, slot].double() - y).abs() <= tol).all(), f"k of {b}"
                assert torch.equal(s.v[page, :, slot], x)
        written[page, slot] = True
        at += n
    for i, (now, old) in enumerate(zip(held, before)):              # every other slot as it was
        now = now.view(torch.uint8) if q8 else now
        if i < 2:
            assert torch.equal(now.transpose(1, 2)[~written], old.transpose(1, 2)[~written])
        else:
            assert torch.equal(now.permute(0, 3, 1, 2)[~written], old.permute(0, 3, 1, 2)[~written])
    if ragged:
        assert (out[at:] == 5.0).all()
    # without queries: the same entries; twice: the same
    mine = [t.view(torch.uint8).clone() if q8 else t.clone() for t in held]
    for t, old in zip(held, before):
        (t.view(torch.uint8) if q8 else t).copy_(old)
    assert paged_append(k, v, s.cache, s.table, s.lens, starts=starts, rotary=rot, norm=hn, positions=given) is None
    for t, m in zip(held, mine):
        assert torch.equal(t.view(torch.uint8) if q8 else t, m)


def test_rows_at_the_ends_of_the_range():
    """Rows of zeros, of the smallest and largest numbers, at the borders of a scale, and not finite ones."""
    from grammar.paged import QuantizedPagedCache, paged_append, paged_read
    dev = _cuda()
    for dt in (torch.float16, torch.bfloat16):
        f = torch.finfo(dt)
        rows = torch.zeros(64, 64, dtype=dt)
        g = torch.Generator("cpu").manual_seed(4)
        rows[1:40] = torch.randn(39, 64, generator=g).to(dt)
        rows[1, 0], rows[2, 5], rows[3, :2] = f.max, -f.max, torch.tensor([f.tiny, -f.tiny])
        rows[4] = 0
        rows[4, 9] = f.smallest_normal * 2.0 ** (-6 if dt == torch.bfloat16 else -9)      # a subnormal number
        for i, x in enumerate((448.0, 449.0, 450.0, 1.75, 1.7578125 if dt == torch.bfloat16 else 1.7509765625, 3.5, 61440.0, 61504.0)):
            rows[5 + i].clamp_(-1, 1)
            rows[5 + i, i] = x
        rows[20, 3], rows[21, 3], rows[22, 63] = float("inf"), float("nan"), -float("inf")
        x = rows.to(dev).view(1, 1, 64, 64)
        cache = QuantizedPagedCache.empty(4, 1, 16, 64, dt, device=dev)
        cache.scales.view(torch.uint8).fill_(7)
        table = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
        lens = torch.tensor([64], dtype=torch.int32, device=dev)
        paged_append(x, x.flip(3).contiguous(), cache, table, lens)
        odd = ~x.isfinite().all(-1)[0, 0]
        want, scale = _quantised(torch.where(odd[:, None], torch.zeros_like(x), x), dt)
        for i, (q, w) in enumerate(((cache.k, want), (cache.v, want.view(torch.uint8).flip(3).view(E4M3)))):
            q, w, sb = q.view(64, 64), w.view(64, 64), cache.scales.view(torch.uint8)[:, 0, i].flatten()
            assert torch.equal(sb[~odd], scale.view(torch.uint8).flatten()[~odd]) and (sb[odd] == 255).all()
            assert torch.equal(q.float()[~odd], w.float()[~odd]) and q.float()[odd].isnan().all()
        k, v = paged_read(cache, table, lens, 64)
        assert k[0, 0][~odd].isfinite().all() and k[0, 0][odd].isnan().all() and torch.equal(k.nan_to_num(), v.flip(3).nan_to_num())
        # appended again, what was read back is what it was
        again = QuantizedPagedCache.empty(4, 1, 16, 64, dt, device=dev)
        paged_append(k, v, again, table, lens)
        k2, v2 = paged_read(again, table, lens, 64)
        assert torch.equal(k.nan_to_num(), k2.nan_to_num()) and torch.equal(v.nan_to_num(), v2.nan_to_num())


def test_append_in_place_queries_and_nowhere_to_put_them():
    from grammar.norm import HeadNorm
    from grammar.paged import paged_append
    from grammar.rotary import Rotary
    s = Setup8([40, 40, 40], 2, 16, 64, "fp16", seed=3)
    rot, norm = Rotary(64, device=s.dev), HeadNorm(1 + 0.1 * torch.randn(64, device=s.dev))
    q, k, v = s.randn(3, 4, 1, 64), s.randn(3, 2, 1, 64), s.randn(3, 2, 1, 64)
    want = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot, norm=norm)
    assert torch.equal(paged_append(k, v, s.cache, s.table, s.lens, q=q, norm=norm), _unturned(q, norm))
    got = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot, norm=norm, out=q)
    assert got is q and torch.equal(q, want)
    s.table[0, 2], s.table[1, 2] = -1, s.k.shape[0]                # pages that do not exist; a place behind the table
    s.lens[2] = 10_000
    held = [t.view(torch.uint8) for t in (s.cache.k, s.cache.v, s.cache.scales)]
    before = [t.clone() for t in held]
    paged_append(s.randn(3, 2, 1, 64), s.randn(3, 2, 1, 64), s.cache, s.table, s.lens, rotary=rot)
    assert all(torch.equal(a, b) for a, b in zip(held, before))
    for starts in ([4, 9, 9, 9], [-4, -1, 7, 100], [9, 9, 9, 9]):   # starts out of the batch
        paged_append(s.randn(6, 2, 64), s.randn(6, 2, 64), s.cache, s.table, s.lens, rotary=rot, norm=norm,
                     starts=torch.tensor(starts, dtype=torch.int32, device=s.dev))
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, before))


def _unturned(q, norm):
    """norm_rotary at position 0, which turns nothing."""
    from grammar.norm import norm_rotary_fwd
    from grammar.rotary import Rotary
    return norm_rotary_fwd(q, None, torch.zeros(q.shape[2], dtype=torch.int32, device=q.device), Rotary(64, device=q.device), norm)[0]


# ---- reading back ----------------------------------------------------------------

@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,Hkv,S", [(64, 3, 16), (128, 1, 64), (128, 9, 16), (64, 40, 32)])
def test_read(q8, dtype, D, Hkv, S):
    from grammar.paged import paged_read
    lens = [0, 1, 15, 16, 17, 100, 333, 64, -3]
    print(f"[case] read q8={q8} {dtype} D{D} Hkv{Hkv} S{S}", flush=True)
    s = (Setup8 if q8 else Setup)(lens, Hkv, S, D, dtype, seed=D + Hkv)
    s.table[6, 2], s.table[5, 0], s.table[7, 0] = -1, s.k.shape[0], 2 ** 31 - 1       # pages that do not exist

    def want(b, x, n):
        k, ok = s.keys(b, x)
        full = torch.zeros(Hkv, n, D, dtype=torch.float64, device=s.dev)
        m = min(n, k.shape[1])
        full[:, :m] = torch.where(ok[None, :m, None], k[:, :m], torch.zeros_like(k[:, :m]))
        return full
    for length in (333, 40, 500, 1):
        got = paged_read(s.cache, s.table, s.lens, length)
        for x, y in zip(got, (s.k, s.v)):
            assert x.dtype == s.dtype and torch.equal(x.double(), torch.stack([want(b, y, length) for b in range(len(lens))]))
    # packed: rows of each sequence, some with room behind their keys, some cut short, some with none, and rows of none
    sizes = [0, 3, 15, 16, 17, 120, 300, 64, 2]
    at = [5 + sum(sizes[:b]) for b in range(len(sizes) + 1)]
    starts = torch.tensor(at, dtype=torch.int32, device=s.dev)
    rows = at[-1] + 7
    wide = torch.full((rows, Hkv + 2, D), 5.0, dtype=s.dtype, device=s.dev)
    k_out, v_out = wide[:, 1:-1], torch.full((rows, Hkv, D), 5.0, dtype=s.dtype, device=s.dev)
    got = paged_read(s.cache, s.table, s.lens, starts=starts, k_out=k_out, v_out=v_out)
    assert got[0] is k_out and got[1] is v_out
    for x, y in zip(got, (s.k, s.v)):
        for b, n in enumerate(sizes):
            assert torch.equal(x[at[b]:at[b + 1]].double().transpose(0, 1), want(b, y, n))
        assert (x[:5] == 5.0).all() and (x[at[-1]:] == 5.0).all()
    assert (wide[:, 0] == 5.0).all() and (wide[:, -1] == 5.0).all()
    out = torch.full_like(v_out, 5.0)
    other = torch.full_like(v_out, 5.0)
    bad = torch.tensor([0, 3, -2, 9, 9, 4, rows + 1, rows + 2, 8, 7], dtype=torch.int32, device=s.dev)
    paged_read(s.cache, s.table, s.lens, starts=bad, k_out=out, v_out=other)           # out of order, out of the batch
    assert (out[9:] == 5.0).all() and (other[9:] == 5.0).all()


# ---- together --------------------------------------------------------------------

def test_serving_run_matches_full_attention():
    """Two conversations as a server runs them, normed, rotated and quantised: prompts in chunks, one joining late, then
    decode steps, packed with a padded batch; every token's result against causal attention in 64 bits over what the
    cache holds; then read back as dense tensors for the training attention."""
    from grammar.attention import flash_attention_fwd
    from grammar.norm import HeadNorm
    from grammar.paged import QuantizedPagedCache, paged_append, paged_attention, paged_read
    from grammar.rotary import Rotary
    dev = _cuda()
    Hq, Hkv, D, S, W = 8, 2, 128, 16, 12
    rot = Rotary(D, device=dev)
    g = torch.Generator("cpu").manual_seed(6)
    norm = HeadNorm(*((1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(dev) for _ in range(2)))
    total = [150, 97]
    x = [torch.randn((n, Hq + 2 * Hkv, D), generator=g).bfloat16().to(dev) for n in total]
    cache = QuantizedPagedCache.empty(2 * W, Hkv, S, D, torch.bfloat16, device=dev)
    for t in (cache.k, cache.v, cache.scales):
        t.view(torch.uint8).fill_(255)
    table = torch.randperm(2 * W, generator=g).int().view(2, W).to(dev)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    starts = torch.zeros(3, dtype=torch.int32, device=dev)
    rows, got = 80, [torch.empty((n, Hq, D), device=dev, dtype=torch.bfloat16) for n in total]
    turned = [torch.empty_like(t) for t in got]
    done = [0, 0]
    for step in [(64, 0), (64, 10), (0, 70)] + [(1, 1)] * 17 + [(1, 0)] * 5:
        packed = torch.full((rows, Hq + 2 * Hkv, D), float("nan"), device=dev, dtype=torch.bfloat16)
        at = 0
        for b, n in enumerate(step):
            packed[at:at + n] = x[b][done[b]:done[b] + n]
            at += n
        starts.copy_(torch.tensor([0, step[0], at], dtype=torch.int32))
        lens.copy_(torch.tensor([done[b] + step[b] for b in range(2)], dtype=torch.int32))
        q, k, v = packed.split([Hq, Hkv, Hkv], 1)
        q = paged_append(k, v, cache, table, lens, starts=starts, q=q, rotary=rot, norm=norm)
        o = paged_attention(q, cache, table, lens, starts=starts)
        at = 0
        for b, n in enumerate(step):
            got[b][done[b]:done[b] + n] = o[at:at + n]
            turned[b][done[b]:done[b] + n] = q[at:at + n]
            done[b] += n
            at += n
    assert done == total
    kd, vd = paged_read(cache, table, lens, 256)
    for b, n in enumerate(total):
        q, k, v = x[b].split([Hq, Hkv, Hkv], 1)
        pos = torch.arange(n, device=dev)
        y, size = _rotated(_normed(k, norm.k_weight, norm.eps)[0], pos, rot)
        page, slot = table[b].long()[pos // S], pos % S
        sc = cache.scales.view(torch.uint8)[page, :, :, slot]
        kq, vq = (t.view(torch.uint8)[page, :, slot].view(E4M3) for t in (cache.k, cache.v))
        _check_rows(kq, sc[:, :, 0], y, _size(y, size), FWD, torch.bfloat16, f"keys of {b}")
        assert torch.equal(vq.float(), _quantised(v, torch.bfloat16)[0].float())
        k, v = (_dequantised(t, sc[:, :, i].contiguous().view(E8M0)) for i, t in enumerate((kq, vq)))
        for dense, t in ((kd, k), (vd, v)):
            assert torch.equal(dense[b, :, :n].transpose(0, 1).double(), t) and not dense[b, :, n:].any()
        k, v = (t.repeat_interleave(Hq // Hkv, 1).transpose(0, 1).contiguous() for t in (k, v))
        w = torch.matmul(turned[b].double().transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(D)
        p = torch.softmax(w.masked_fill(torch.ones(n, n, dtype=torch.bool, device=dev).triu(1), -math.inf), -1)
        o, sz = torch.matmul(p, v), torch.matmul(p, v.abs())
        # (P in bf16, and e of scores whose A is at most 20)
        tol = lambda o, sz: (2.0 ** -8 + 2.0 ** -24 * 136 * 20) * (sz + 2 * o.abs()) * 1.01 + 2.0 ** -100  # noqa: E731
        assert ((got[b].double() - o.transpose(0, 1)).abs() <= tol(o, sz).transpose(0, 1)).all(), f"conversation {b}"
        assert float(torch.matmul(turned[b].double().abs().transpose(0, 1), k.abs().transpose(1, 2).contiguous()).max()) <= 20 * math.sqrt(D)
        # the dense keys and values through the training attention (causal, as many queries as keys: zeros behind)
        qd = torch.zeros(1, Hq, 256, D, dtype=torch.bfloat16, device=dev)
        qd[0, :, :n] = turned[b].transpose(0, 1)
        dense = flash_attention_fwd(qd, *(t[b:b + 1].repeat_interleave(Hq // Hkv, 1) for t in (kd, vd)), causal=True)
        assert ((dense[0, :, :n].double() - o).abs() <= tol(o, sz)).all(), f"dense attention of {b}"


def test_bound_steps_on_streams_and_in_graphs():
    """A decode loop on fixed buffers: bound once, captured, replayed as the lengths grow; two graphs, each with its own
    binding; calls on another stream."""
    from grammar.norm import HeadNorm
    from grammar.paged import bind_paged_append, bind_paged_attention, paged_append, paged_attention, paged_read
    from grammar.rotary import Rotary
    s = Setup8([400, 3000], 2, 16, 128, "bf16", seed=12, width=200, spare=40)
    free = s.unused
    for b, have in ((0, 25), (1, 188)):
        for i in range(3):
            s.table[b, have + i] = free.pop()
    rot, norm = Rotary(128, device=s.dev), HeadNorm(*(1 + 0.2 * torch.randn(128, device=s.dev) for _ in range(2)))
    q, k, v = s.randn(2, 8, 1, 128), s.randn(2, 2, 1, 128), s.randn(2, 2, 1, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            add, qr = bind_paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot, norm=norm, stream=side)
            attend, o = bind_paged_attention(qr, s.cache, s.table, s.lens, stream=side)
            add()
            attend()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                s.lens.add_(1)
                add()
                attend()
                back = paged_read(s.cache, s.table, s.lens, 600)
            graphs.append((graph, qr, o, add, attend, back))
    torch.cuda.synchronize()
    s.lens.copy_(torch.tensor([400, 3000], dtype=torch.int32))
    for i in range(8):
        graph, qr, o, _, _, back = graphs[i % 2]
        for t in (q, k, v):
            t.copy_(s.randn(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        s.lens_host = [401 + i, 3001 + i]
        assert s.lens.tolist() == s.lens_host
        kept = [t.view(torch.uint8).clone() for t in (s.cache.k, s.cache.v, s.cache.scales)]
        want = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot, norm=norm)
        assert torch.equal(want, qr)
        assert all(torch.equal(t.view(torch.uint8), m) for t, m in zip((s.cache.k, s.cache.v, s.cache.scales), kept))
        eager = paged_attention(want, s.cache, s.table, s.lens)
        assert torch.equal(eager, o)
        assert all(torch.equal(a, b) for a, b in zip(paged_read(s.cache, s.table, s.lens, 600), back))
        sc = s.cache.scales.view(torch.uint8)
        s.k, s.v = (_dequantised(t, sc[:, :, j].contiguous().view(E8M0)).to(s.dtype) for j, t in enumerate((s.cache.k, s.cache.v)))
        for b in range(2):
            ref, _, size = _attention(s, b, qr[b].transpose(0, 1))
            _check(o[b].transpose(0, 1), ref, size, qr[b].transpose(0, 1), s, b, f"replay {i}")
    for stream in (side, side.cuda_stream):
        side.wait_stream(torch.cuda.current_stream())
        got = paged_attention(want, s.cache, s.table, s.lens, stream=stream)
        back2 = paged_read(s.cache, s.table, s.lens, 600, stream=stream)
        side.synchronize()
        assert torch.equal(got, eager) and all(torch.equal(a, b) for a, b in zip(back, back2))


def test_a_binding_keeps_its_weights():
    """Weights that a norm gets after a call was bound are not the binding's, and those it was bound with stay."""
    import gc
    import weakref
    from grammar.norm import HeadNorm
    from grammar.paged import bind_paged_append, paged_append
    s = Setup8([20, 33], 2, 16, 64, "bf16", seed=3)
    q, k = s.randn(2, 4, 3, 64), s.randn(2, 2, 3, 64)
    norm = HeadNorm(*(1 + 0.2 * torch.randn(64, device=s.dev) for _ in range(2)))
    want = paged_append(k, k, s.cache, s.table, s.lens, q=q, norm=norm)
    add, out = bind_paged_append(k, k, s.cache, s.table, s.lens, q=q, norm=norm)
    held = [weakref.ref(w) for w in (norm.q_weight, norm.k_weight)]
    norm.q_weight = norm.k_weight = None
    gc.collect()
    assert all(w() is not None for w in held)
    add()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_calls_of_two_threads_at_once():
    import threading
    from grammar.paged import paged_append, paged_attention
    from grammar.rotary import Rotary
    rot = Rotary(128, device=torch.device("cuda:0"))
    sides = [torch.cuda.Stream() for _ in range(2)]
    cases = []
    for i in range(2):
        s = Setup8([4000 + 900 * i, 70, 2500], 2, 16, 128, "bf16", seed=20 + i, width=400)
        q, k, v = s.randn(3, 8, 5, 128), s.randn(3, 2, 5, 128), s.randn(3, 2, 5, 128)
        qr = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot)
        cases.append((s, q, k, v, qr, paged_attention(qr, s.cache, s.table, s.lens)))
    torch.cuda.synchronize()
    got, errors, start = [[], []], [], threading.Barrier(2)

    def loop(i):
        try:
            s, q, k, v, *_ = cases[i]
            start.wait(30)
            with torch.cuda.stream(sides[i]):
                for _ in range(40):
                    qr = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot)
                    got[i].append((qr, paged_attention(qr, s.cache, s.table, s.lens)))
        except Exception as e:                                   # shown below: a thread's own would be lost
            errors.append(e)
    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not errors
    for (*_, qr, o), results in zip(cases, got):
        assert len(results) == 40 and all(torch.equal(a, qr) and torch.equal(b, o) for a, b in results)


def test_caches_can_be_copied_and_pickled():
    import copy
    import pickle
    from grammar.paged import QuantizedPagedCache, paged_append, paged_attention
    s = Setup8([40, 50], 2, 16, 64, "fp16", seed=6)
    q, k, v = s.randn(2, 4, 1, 64), s.randn(2, 2, 1, 64), s.randn(2, 2, 1, 64)
    for make in (copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        c = make(s.cache)
        assert type(c) is QuantizedPagedCache and c.desc.k == c.k.data_ptr() != s.cache.k.data_ptr() and c.dtype == s.dtype
        old = s.cache.k.view(torch.uint8).clone()
        paged_append(k, v, c, s.table, s.lens)
        assert torch.equal(s.cache.k.view(torch.uint8), old)       # the copy's pages are its own
        there = make(s.cache)
        paged_append(k, v, there, s.table, s.lens)
        assert torch.equal(paged_attention(q, there, s.table, s.lens), paged_attention(q, c, s.table, s.lens))


def test_outputs_share_memory_with_their_own_input_only():
    from grammar import runtime as rt
    from grammar.paged import paged_append, paged_attention, paged_read
    from grammar.rotary import Rotary
    s = Setup8([40, 50, 300], 2, 16, 64, "fp16", seed=7)
    rot = Rotary(64, device=s.dev)
    starts = torch.tensor([0, 9, 18, 27], dtype=torch.int32, device=s.dev)
    rows = s.randn(27, 14, 64)
    q, k, v = rows[:, :8], rows[:, 8:10], rows[:, 10:12]
    args = (s.cache, s.table, s.lens)
    inside = [t.view(torch.uint8).view(-1).view(torch.float16)[:2 * 2 * 64].view(2, 2, 64) for t in (s.cache.k, s.cache.scales)]
    two = torch.tensor([0, 1, 2, 2], dtype=torch.int32, device=s.dev)
    for bad in (lambda: paged_append(k, v, *args, starts=starts, q=q, rotary=rot, out=rows[:, 4:12]),
                lambda: paged_append(k[:2], v[:2], *args, starts=two, q=q[:2, :2], rotary=rot, out=inside[0]),
                lambda: paged_append(k[:2], v[:2], *args, starts=two, q=q[:2, :2], rotary=rot, out=inside[1]),
                lambda: paged_attention(q, *args, starts=starts, out=rows[:, 6:14]),
                lambda: paged_attention(q[:2, :2], *args, starts=two, out=inside[0]),
                lambda: paged_attention(q[:2, :2], *args, starts=two, out=inside[1]),
                lambda: paged_read(*args, starts=two, k_out=inside[0], v_out=torch.empty_like(inside[0])),
                lambda: paged_read(*args, starts=two, k_out=torch.empty_like(inside[0]), v_out=inside[1]),
                lambda: paged_read(*args, starts=starts, k_out=rows[:, :2], v_out=rows[:, 1:3])):
        before = rows.clone(), s.cache.k.view(torch.uint8).clone(), s.cache.scales.view(torch.uint8).clone()
        with pytest.raises(rt.GrError, match="shares? memory"):
            bad()
        assert torch.equal(rows, before[0]) and torch.equal(s.cache.k.view(torch.uint8), before[1])
        assert torch.equal(s.cache.scales.view(torch.uint8), before[2])
    paged_read(*args, starts=starts, k_out=rows[:, :2], v_out=rows[:, 2:4])
    # attention in place: in tiles of 32, 64 and 128 rows, a workgroup a tile and shared out
    for m, lens, width in ((1, [40, 50, 3000], None), (9, [40, 50, 300], None), (150, [150, 500, 4000], None),
                           (1, [40, 50, 3000], 2048), (150, [150, 500, 4000], 2048)):
        t = Setup8(lens, 2, 16, 64, "fp16", seed=m, width=width)
        x = t.randn(3, 8, m, 64)
        o = paged_attention(x, t.cache, t.table, t.lens)
        assert paged_attention(x, t.cache, t.table, t.lens, out=x) is x and torch.equal(x, o)


def test_refusals():
    from grammar import runtime as rt
    from grammar.norm import HeadNorm
    from grammar.paged import QuantizedPagedCache, paged_append, paged_attention, paged_read
    from grammar.rotary import Rotary
    s = Setup8([20, 20], 2, 16, 64, "fp16")
    rot = Rotary(64, device=s.dev)
    q, k, w = s.randn(2, 4, 1, 64), s.randn(2, 2, 1, 64), torch.ones(64, device=s.dev)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=s.dev)
    kq, sc = s.cache.k, s.cache.scales

    def make(k=kq, v=kq, scales=sc, dtype=torch.float16):
        return QuantizedPagedCache(k, v, scales, dtype)

    def append(k=k, v=k, **kw):
        return paged_append(k, v, s.cache, s.table, s.lens, **kw)

    def read(*a, **kw):
        return paged_read(s.cache, s.table, s.lens, *a, **kw)
    for bad in (lambda: make(k=s.k), lambda: make(v=kq[:1]), lambda: make(scales=sc[:, :, :1]), lambda: make(scales=sc.view(torch.uint8)),
                lambda: make(dtype=torch.float32), lambda: make(k=kq[..., :32], v=kq[..., :32]), lambda: make(k=kq.cpu()),
                lambda: make(scales=sc.cpu()), lambda: make(k=kq[:1].expand(*kq.shape)), lambda: make(scales=sc[:1].expand(*sc.shape)),
                lambda: make(k=kq[:, :, :8], v=kq[:, :, :8], scales=sc[..., :8]), lambda: make(scales=sc[..., ::2]),
                lambda: append(k=k.bfloat16(), v=k.bfloat16()), lambda: append(q=q), lambda: append(out=q),
                lambda: append(q=q, norm=HeadNorm(w.bfloat16())), lambda: append(q=q, norm=HeadNorm(w[:32])),
                lambda: append(q=q, norm=HeadNorm(w), positions=s.lens), lambda: paged_attention(q.bfloat16(), s.cache, s.table, s.lens),
                lambda: paged_read(s.cache, s.table[0], s.lens, 5), lambda: paged_read(s.cache, s.table[0, 0], s.lens, 5),
                lambda: paged_read(s.cache, s.table, s.lens[:1], 5), lambda: read(), lambda: read(-1), lambda: read(starts=starts), lambda: read(10, starts=starts),
                lambda: read(k_out=s.randn(2, 2, 20, 64)), lambda: read(20, k_out=s.randn(2, 2, 21, 64), v_out=s.randn(2, 2, 21, 64)),
                lambda: read(k_out=s.randn(2, 3, 20, 64), v_out=s.randn(2, 3, 20, 64)),
                lambda: read(k_out=s.randn(2, 2, 20, 64).bfloat16(), v_out=s.randn(2, 2, 20, 64).bfloat16()),
                lambda: read(k_out=s.randn(2, 2, 20, 64), v_out=s.randn(2, 2, 1, 64).expand(2, 2, 20, 64)),
                lambda: read(k_out=s.randn(2, 2, 20, 64), v_out=s.randn(2, 2, 19, 64))):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros(4, 2, 16, 72, dtype=torch.uint8, device=s.dev).view(E4M3)[..., :64]        # rows 72 bytes apart
    cache = QuantizedPagedCache(wide, wide.clone(memory_format=torch.preserve_format), sc[:4], torch.float16)
    for bad in (lambda: paged_append(k, k, cache, s.table, s.lens), lambda: paged_attention(q, cache, s.table, s.lens),
                lambda: paged_read(cache, s.table, s.lens, 5)):
        with pytest.raises(rt.GrError, match="multiples of 16"):
            bad()
    assert paged_attention(q[:, :, :0], s.cache, s.table, s.lens).shape == (2, 4, 0, 64)
    assert append(k=k[:, :, :0], v=k[:, :, :0]) is None and read(0)[0].shape == (2, 2, 0, 64)
