"""The paged key/value cache: appending (gr_paged_append) and attention over it
(gr_paged_attn) against the definitions in 64 bits, at the lengths, masks, pages
and layouts where they can go wrong."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


class Setup:
    """A cache with its pages in no order, sequences of `lens` keys, and random
    entries in every slot, live or stale."""

    def __init__(self, lens, Hkv, S, D, dtype, seed=0, spare=3, width=None):
        from grammar.paged import PagedCache
        dev = _cuda()
        g = torch.Generator("cpu").manual_seed(seed)
        need = [-(-max(0, m) // S) for m in lens]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).int()
        self.width = width or max(1, max(need))
        table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        at = 0
        for b, p in enumerate(need):
            table[b, :p] = order[at:at + p]
            at += p
        self.unused = order[at:].tolist()
        self.table, self.lens_host, self.S, self.D, self.Hkv = table.to(dev), list(lens), S, D, Hkv
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        shape = (total, Hkv, S, D)
        self.k, self.v = (torch.randn(shape, generator=g).to(DT[dtype]).to(dev) for _ in range(2))
        self.cache = PagedCache(self.k, self.v)
        self.g, self.dev, self.dtype = g, dev, DT[dtype]

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g).to(self.dtype).to(self.dev)

    def keys(self, b, x):
        """The sequence's keys (x: self.k or self.v), [Hkv, len, D] in 64 bits, and which of them exist."""
        m, S, P = max(0, self.lens_host[b]), self.S, self.k.shape[0]
        m = min(m, self.width * S)
        j = torch.arange(m, device=self.dev)
        page = self.table[b].long()[j // S] if m else j
        ok = (page >= 0) & (page < P)
        return x[page.clamp(0, P - 1), :, j % S].double().transpose(0, 1).contiguous(), ok


def _attention(s, b, q, causal=True, scale=None):
    """q [n, Hq, D] of sequence b -> (o, lse, sum p|v| / l), [n, Hq, ..] in 64 bits; a row without keys 0 and -inf."""
    n, Hq, D = q.shape
    k, ok = s.keys(b, s.k)
    v, _ = s.keys(b, s.v)
    G, m = Hq // s.Hkv, k.shape[1]
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    sc = torch.matmul(q.double().transpose(0, 1), k.transpose(1, 2).contiguous()) * (scale or 1 / math.sqrt(D))
    hide = ~ok[None, :].expand(n, m)
    if causal:
        place = s.lens_host[b] - n + torch.arange(n, device=s.dev)
        hide = hide | (torch.arange(m, device=s.dev)[None] > place[:, None])
    sc = sc.masked_fill(hide, float("-inf"))
    lse = torch.logsumexp(sc, -1) if m else torch.full((Hq, n), -math.inf, dtype=torch.float64, device=s.dev)
    p = torch.exp(sc - lse[..., None]).masked_fill(hide, 0.0)
    # what no row may see does not count, NaN or not
    live = ~hide
    o = torch.zeros((Hq, n, D), dtype=torch.float64, device=s.dev)
    size = torch.zeros_like(o)
    if m:
        clean = torch.where(v.isfinite(), v, torch.zeros_like(v))
        o, size = torch.matmul(p, clean), torch.matmul(p, clean.abs())
        for h, j in (~v.isfinite()).any(-1).nonzero().tolist():        # each such key to the rows that see it
            rows = live[:, j]
            o[h, rows] += p[h, rows, j, None] * torch.where(v[h, j].isfinite(), torch.zeros_like(v[h, j]), v[h, j])
    return o.transpose(0, 1), lse.transpose(0, 1), size.transpose(0, 1)


def _check(got, want, size, what, extra=0.0):
    """The result rounds once (half a step of |o|); P rounds to the type before
    the product, half a step of each p in the sum of p v (size) and in the sum of
    p (|o|); scores in fp32 are off by 2^-24 of a sum of D products a few times
    over: at most 2e-4 of size at these inputs."""
    u = torch.finfo(got.dtype).eps / 2
    tol = (u * (size + 2 * want.abs()) + 2e-4 * size) * 1.01 + 2.0 ** -24 + extra
    bad = ~((got.double() - want).abs() <= tol) & want.isfinite()
    bad |= want.isnan() != got.isnan()
    bad |= want.isinf() & (got.double() != want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() - tol).max())}"


def _check_lse(got, want, dtype, what):
    # l is summed from p rounded to the type, half a step each; the scores as above
    tol = torch.finfo(dtype).eps / 2 * 1.01 + 2e-4
    none = want == -math.inf
    assert torch.equal(got == -math.inf, none), what
    assert ((got.double() - want).abs()[~none] <= tol).all(), what


def _run(s, news, Hq, causal=True, ragged=False, pad=0, scale=None, workspace=None, hints=True, strided=False):
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
    got = paged_attention(q, s.cache, s.table, s.lens, starts=starts, causal=causal, scale=scale, out=out, lse=lse,
                          workspace=workspace, **more)
    torch.cuda.synchronize()
    assert got is out
    row = 0
    for b, n in enumerate(news):
        qb = q[row:row + n] if ragged else q[b].transpose(0, 1)
        ob = out[row:row + n] if ragged else out[b].transpose(0, 1)
        lb = lse[row:row + n] if ragged else lse[b]
        o, ls, size = _attention(s, b, qb, causal, scale)
        _check(ob, o, size, f"sequence {b}: {n} tokens, {s.lens_host[b]} keys")
        if o.isfinite().all():
            _check_lse(lb, ls, s.dtype, f"lse of sequence {b}")
        row += n
    if ragged:
        assert (out[row:] == 5.0).all() and (lse[row:] == 7.0).all()      # rows behind the last sequence
    return out


LENS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 257, 1000, 0]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,Hkv,S", [(1, 3, 16), (4, 2, 16), (7, 1, 64), (16, 1, 32), (40, 1, 16), (70, 1, 128)])
def test_single_tokens(dtype, D, G, Hkv, S):
    print(f"[case] decode {dtype} D{D} G{G} Hkv{Hkv} S{S}", flush=True)
    s = Setup(LENS, Hkv, S, D, dtype, seed=G)
    _run(s, [1] * len(LENS), G * Hkv)
    _run(s, [1] * len(LENS), G * Hkv, ragged=True, pad=3, hints=False, strided=True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G,Hkv", [(2, 1, 2), (5, 7, 1), (13, 5, 2), (33, 1, 2), (64, 2, 1), (100, 3, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_few_tokens(dtype, D, n, G, Hkv, causal):
    """Lengths below, at and above the new tokens' count: with fewer keys than new tokens some rows see nothing."""
    lens = [n, n + 1, n + 16, max(0, n - 3), 0, 1, 3 * n + 70, 513]
    print(f"[case] few {dtype} D{D} n{n} G{G} causal={causal}", flush=True)
    s = Setup(lens, Hkv, 16, D, dtype, seed=n)
    _run(s, [n] * len(lens), G * Hkv, causal=causal, strided=True)


@pytest.mark.parametrize("dtype,D,G,Hkv,S", [("bf16", 128, 4, 2, 16), ("fp16", 64, 1, 4, 32), ("bf16", 64, 6, 1, 128),
                                             ("fp16", 128, 3, 2, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_mixed_batches(dtype, D, G, Hkv, S, causal):
    """Prompts' chunks among single tokens and sequences with nothing new, packed and padded."""
    news = [1, 0, 150, 1, 7, 0, 1, 301, 1, 0]
    lens = [40, 99, 150, 700, 7, 0, 1, 900, 0, 5]
    print(f"[case] mixed {dtype} D{D} G{G} Hkv{Hkv} S{S} causal={causal}", flush=True)
    s = Setup(lens, Hkv, S, D, dtype, seed=D + G)
    _run(s, news, G * Hkv, causal=causal, ragged=True, pad=9)
    _run(s, news, G * Hkv, causal=causal, ragged=True, hints=False)


def test_more_sequences_than_a_wave_has_lanes():
    rng = random.Random(3)
    news = [rng.choice((0, 1, 1, 1, 3, 40)) for _ in range(150)]
    lens = [n + rng.choice((0, 0, 1, 30, 200)) for n in news]
    s = Setup(lens, 2, 16, 64, "bf16", seed=4)
    _run(s, news, 6, ragged=True, pad=2)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64)])
def test_whole_prompts(dtype, D):
    print(f"[case] prompts {dtype} D{D}", flush=True)
    s = Setup([1111, 400], 2, 64, D, dtype, seed=8)
    _run(s, [1111, 130], 8, ragged=True)


def _needs_workspace(s, rows, Hq, starts=None):
    import ctypes
    from grammar import runtime as rt
    batch = rt.PagedBatch(s.table.data_ptr(), s.width, s.lens.data_ptr(), starts, len(s.lens_host), rows, s.width, 0, 0)
    return int(rt.lib().gr_paged_attn_workspace(s.cache.ref, ctypes.addressof(batch), Hq))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G,Hkv", [(1, 4, 2), (1, 1, 3), (5, 7, 1), (3, 20, 1), (50, 4, 1)])
def test_shared_work_of_ragged_lengths(dtype, D, n, G, Hkv):
    """A table with room for long contexts, so that the work is shared out, over short, empty and long sequences:
    shares that end in a tile's first, last and only blocks, and tiles of one share and of many."""
    lens = [m + n - 1 for m in LENS] + [0, 3000, 64, 128, 5000, n]
    s = Setup(lens, Hkv, 16, D, dtype, seed=n, width=1024)
    print(f"[case] shared {dtype} D{D} n{n} G{G} Hkv{Hkv}", flush=True)
    assert _needs_workspace(s, n, G * Hkv) > 0
    _run(s, [n] * len(lens), G * Hkv, hints=False, strided=True)


@pytest.mark.parametrize("dtype,D,G,Hkv", [("bf16", 128, 4, 2), ("fp16", 64, 1, 2)])
def test_shared_mixed_batches(dtype, D, G, Hkv):
    news = [1, 0, 150, 1, 7, 0, 1, 301, 1, 0] + [1] * 70
    lens = [40, 99, 150, 4000, 7, 0, 1, 900, 0, 5] + [3 * i for i in range(70)]
    s = Setup(lens, Hkv, 16, D, dtype, seed=D, width=2048)
    print(f"[case] shared mixed {dtype} D{D} G{G}", flush=True)
    assert _needs_workspace(s, sum(news) + 5, G * Hkv, s.lens.data_ptr()) > 0
    for causal in (True, False):
        _run(s, news, G * Hkv, causal=causal, ragged=True, pad=5, hints=False)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("G,Hkv", [(8, 16), (4, 8)], ids=["many", "few"])
def test_mixed_batches_of_a_workgroup_a_tile(dtype, D, G, Hkv):
    """Grids that fill the GPU and grids that do not (their tiles' keys in two groups), single tokens among them."""
    news = [1, 130, 0, 33, 300, 1, 16] + [1, 0, 2] * 25 + [34]
    lens = [260, 131, 9, 33, 449, 0, 80] + [5 * i for i in range(75)] + [70]
    s = Setup(lens, Hkv, 32, D, dtype, seed=G)
    print(f"[case] tiles {dtype} D{D} G{G} Hkv{Hkv}", flush=True)
    assert _needs_workspace(s, sum(news) + 3, G * Hkv, s.lens.data_ptr()) == 0
    for causal in (True, False):
        _run(s, news, G * Hkv, causal=causal, ragged=True, pad=3, hints=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 40])
def test_long_contexts_share_their_keys_out(D, n):
    """Keys over several workgroups and merged: as many as the default takes, fewer with a smaller workspace, none
    with an empty one; each twice, bit for bit the same."""
    from grammar.paged import paged_attention
    lens = [20_011, 3, 5000]
    s = Setup(lens, 2, 32, D, "bf16", seed=D)
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
            _check(a[i].transpose(0, 1), o, sz, f"workspace {size}, sequence {i}")


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("fp16", 128)])
@pytest.mark.parametrize("n,G", [(1, 4), (9, 4), (70, 2)])
@pytest.mark.parametrize("width", [None, 2048], ids=["tile", "shared"])
def test_hidden_entries_may_hold_anything(dtype, D, n, G, width):
    """Stale slots and pages of other sequences hold NaN; a value that only later tokens see holds inf or NaN, and
    so do they, but no earlier row."""
    lens = [n, n + 7, n + 100, 200 + n]
    s = Setup(lens, 2, 16, D, dtype, seed=n, width=width)
    nan = float("nan")
    live = torch.zeros(s.k.shape[0], s.S, dtype=torch.bool)
    for b, m in enumerate(lens):
        for j in range(m):
            live[int(s.table[b, j // s.S]), j % s.S] = True
    dead = (~live).to(s.dev)[:, None, :, None]
    s.k.masked_fill_(dead, nan)
    s.v.masked_fill_(dead, nan)
    print(f"[case] hidden {dtype} D{D} n{n} width {width}", flush=True)
    assert _run(s, [n] * 4, 2 * G, hints=False).isfinite().all()
    if n == 1:
        return
    # the last token's entries: NaN key in head 0; inf and NaN values in head 1, and a finite huge one
    for b, m in enumerate(lens[:3]):
        page, slot = int(s.table[b, (m - 1) // s.S]), (m - 1) % s.S
        s.k[page, 0, slot, 3] = nan
        s.v[page, 1, slot, 5], s.v[page, 1, slot, D - 1] = float("inf"), nan
    out = _run(s, [n] * 4, 2 * G, hints=False)
    assert out[:3, :, :-1].isfinite().all()                     # earlier rows
    assert out[:3, :G, -1].isnan().all() and out[:3, G:, -1, 5].isinf().all() and out[:3, G:, -1, D - 1].isnan().all()


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("G,Hkv", [(8, 24), (4, 12)], ids=["many", "few"])
@pytest.mark.parametrize("ragged", [False, True])
def test_hidden_entries_of_chunks(dtype, D, G, Hkv, ragged):
    """The same in tiles of 128 rows (grids that fill the GPU and grids that do not), and pages that do not exist
    at a chunk's start, middle and end."""
    n, S = 90, 16
    lens = [n, n + 7, n + 100, 300 + n]
    s = Setup(lens, Hkv, S, D, dtype, seed=G)
    live = torch.zeros(s.k.shape[0], S, dtype=torch.bool)
    for b, m in enumerate(lens):
        for j in range(m):
            live[int(s.table[b, j // S]), j % S] = True
    dead = (~live).to(s.dev)[:, None, :, None]
    s.k.masked_fill_(dead, float("nan"))
    s.v.masked_fill_(dead, float("nan"))
    for b, m in enumerate(lens):
        page, slot = int(s.table[b, (m - 1) // S]), (m - 1) % S
        s.k[page, 0, slot, 3] = float("nan")
        s.v[page, 1, slot, 5], s.v[page, 1, slot, D - 1] = float("inf"), float("nan")
    s.table[1, 3], s.table[2, 0], s.table[3, 5], s.table[3, 17] = -1, s.k.shape[0], -9, 2 ** 31 - 1
    print(f"[case] hidden chunks {dtype} D{D} G{G} Hkv{Hkv} ragged {ragged}", flush=True)
    out = _run(s, [n] * 4, G * Hkv, ragged=ragged, pad=3 * ragged, hints=False)
    if not ragged:
        assert out[:, :, :-1].isfinite().all() and out[:, 2 * G:].isfinite().all()


@pytest.mark.parametrize("width", [None, 2048], ids=["tile", "shared"])
def test_pages_that_do_not_exist(width):
    """Page ids out of range, keys behind the table and starts out of the batch read nothing."""
    from grammar.paged import paged_attention
    s = Setup([100, 100, 64], 2, 16, 64, "bf16", seed=1, width=width)
    s.table[0, 2], s.table[0, 6], s.table[1, 0] = -1, s.k.shape[0], 2 ** 31 - 1
    s.table[2, :4] = -7
    for n in (1, 20):
        out = _run(s, [n] * 3, 4, hints=False)
        assert not out[2].any()
    s.lens_host[1] = 50_000                                     # more keys than the table holds
    s.lens.copy_(torch.tensor(s.lens_host, dtype=torch.int32))
    _run(s, [1] * 3, 4, hints=False)
    s.lens_host[1] = -5
    s.lens.copy_(torch.tensor(s.lens_host, dtype=torch.int32))
    assert not _run(s, [3] * 3, 4, hints=False)[1].any()
    q = s.randn(6, 4, 64)
    out = torch.full_like(q, 5.0)
    for starts in ([0, 3, 2, 9], [-4, -1, 7, 100], [6, 6, 6, 6]):     # the second has no valid sequence, nor the third
        paged_attention(q, s.cache, s.table, s.lens, starts=torch.tensor(starts, dtype=torch.int32, device=s.dev), out=out)
        torch.cuda.synchronize()
        assert (out[3:] == 5.0).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_growing_scores_and_other_scales(dtype):
    """Keys whose scores rise along the sequence by hundreds of powers of two, and scales above 1."""
    s = Setup([700, 300], 2, 16, 64, dtype, seed=2)
    for b, m in enumerate(s.lens_host):
        j = torch.arange(m, device=s.dev)
        page = s.table[b].long()[j // s.S]
        s.k[page, :, j % s.S] = (s.k[page, :, j % s.S].float() * (1 + j[:, None, None] / 10)).to(s.dtype)
    # exact in the limit of one key: scores differ by tens; a score's fp32 error grows with it (2^-24 of 64 products
    # of up to 4 x 280: 4e-3 in the exponent), so only inputs whose softmax is nearly one key are used here
    from grammar.paged import paged_attention
    for n, scale in ((1, 1.5), (40, 1.5), (1, 20.0)):
        q = s.randn(2, 4, n, 64)
        got = paged_attention(q, s.cache, s.table, s.lens, scale=scale)
        for b in range(2):
            o, _, size = _attention(s, b, q[b].transpose(0, 1), scale=scale)
            _check(got[b].transpose(0, 1), o, size, f"scale {scale}", extra=2 * 4e-3 * scale * float(size.max()))


def test_cache_layouts_and_table_strides():
    """Pages stored [pages, page_size, heads, D], keys and values in one tensor, and a table that is a slice."""
    from grammar.paged import PagedCache, paged_attention
    s = Setup([77, 130, 5], 3, 16, 128, "bf16", seed=9)
    both = torch.stack((s.k.transpose(1, 2), s.v.transpose(1, 2)), 2)        # [pages, S, 2, heads, D]
    both = both.contiguous()
    cache = PagedCache(both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2))
    table = torch.full((3, 40), 10 ** 6, dtype=torch.int32, device=s.dev)
    table[:, 5:5 + s.width] = s.table
    for n in (1, 4, 60):
        q = s.randn(3, 6, n, 128)
        want = paged_attention(q, s.cache, s.table, s.lens)
        assert torch.equal(paged_attention(q, cache, table[:, 5:5 + s.width], s.lens), want)


def test_offsets_past_32_bits():
    """Pages whose elements lie beyond 2^31 of the cache's start."""
    from grammar.paged import PagedCache, paged_append, paged_attention
    dev = _cuda()
    P, H, S, D = 70_000, 4, 64, 128                              # 2.3e9 elements each
    cache = PagedCache.empty(P, H, S, D, torch.bfloat16, device=dev)
    table = torch.tensor([[P - 1, 0, P - 3, 65_537]], dtype=torch.int32, device=dev)
    g = torch.Generator("cpu").manual_seed(1)
    k, v = (torch.randn((1, H, 250, D), generator=g).bfloat16().to(dev) for _ in range(2))
    lens = torch.tensor([250], dtype=torch.int32, device=dev)
    paged_append(k, v, cache, table, lens)
    j = torch.arange(250, device=dev)
    assert torch.equal(cache.k[table[0].long()[j // S], :, j % S].transpose(0, 1), k[0])
    q = torch.randn((1, 8, 250, D), generator=g).bfloat16().to(dev)
    s = Setup([250], H, S, D, "bf16")
    s.k[s.table[0].long()[j // S], :, j % S] = k[0].transpose(0, 1)
    s.v[s.table[0].long()[j // S], :, j % S] = v[0].transpose(0, 1)
    for n in (1, 20, 250):
        a = paged_attention(q[:, :, -n:], cache, table, lens)
        assert torch.equal(a, paged_attention(q[:, :, -n:], s.cache, s.table, s.lens))


# ---- appending -------------------------------------------------------------------

def _rotated(x, pos, rot):
    """x [n, H, D], pos [n] or [axes, n] -> 64 bits, and |x1| + |x2| of each pair."""
    from test_rotary_gpu import _exact
    y, size = _exact(x.transpose(0, 1)[None], pos, rot)
    return y[0].transpose(0, 1), size[0].transpose(0, 1)


def _close(got, want, size, what):
    from test_rotary_gpu import _check as check
    check(got, want, size, what)


APPENDS = [
    # news, lens, Hq, Hkv, D, S, rotary_dim, sections, interleaved, dtype, ragged
    ([1] * 5, [1, 16, 17, 40, 100], 8, 2, 128, 16, 128, None, False, "bf16", False),
    ([1] * 3, [5, 64, 33], 1, 1, 64, 32, 32, None, True, "fp16", False),
    ([9] * 2, [9, 30], 4, 4, 64, 16, 64, [10, 11, 11], False, "fp16", False),
    ([1, 0, 40, 1, 17], [3, 8, 40, 99, 50], 6, 3, 128, 16, 64, None, False, "bf16", True),
    ([300, 2], [310, 2], 32, 8, 128, 64, 128, [16, 24, 24], True, "bf16", True),
    ([500, 1, 60], [700, 90, 60], 32, 8, 128, 16, 128, None, False, "bf16", True),
    ([600, 1, 500], [610, 20, 500], 35, 7, 64, 32, 32, None, False, "fp16", True),
    ([2, 30], [1, 25], 2, 1, 64, 16, 64, None, False, "fp16", True),          # more tokens than keys: places below 0
]


@pytest.mark.parametrize("news,lens,Hq,Hkv,D,S,rd,sections,inter,dtype,ragged", APPENDS)
@pytest.mark.parametrize("given", [False, True])
def test_append(news, lens, Hq, Hkv, D, S, rd, sections, inter, dtype, ragged, given):
    from grammar.paged import paged_append
    from grammar.rotary import Rotary
    print(f"[case] append {news} D{D} S{S} {sections} {dtype} given={given}", flush=True)
    s = Setup(lens, Hkv, S, D, dtype, seed=len(news))
    rot = Rotary(D, rotary_dim=rd, sections=sections, interleaved=inter, device=s.dev)
    pad = 4 if ragged else 0
    T, B = sum(news) + pad, len(news)
    rows = s.randn(T, Hq + 2 * Hkv, D)                            # a projection's rows: q, k, v side by side
    where = rows if ragged else rows.view(B, news[0], Hq + 2 * Hkv, D).transpose(1, 2)
    q, k, v = where.split([Hq, Hkv, Hkv], 1)
    lead = (rot.naxes,) if rot.naxes > 1 else ()
    pos = torch.randint(0, 5000, lead + (T,), generator=s.g, dtype=torch.int32).to(s.dev) if given else None
    starts = torch.tensor([0] + [sum(news[:b + 1]) for b in range(B)], dtype=torch.int32, device=s.dev) if ragged else None
    before = s.k.clone(), s.v.clone()
    out = torch.full_like(q, 5.0)
    got = paged_append(k, v, s.cache, s.table, s.lens, starts=starts, q=q, rotary=rot, out=out,
                       positions=pos if pos is None or ragged else pos.view(lead + (B, news[0])))
    torch.cuda.synchronize()
    assert got is out
    written = torch.zeros(s.k.shape[0], S, dtype=torch.bool, device=s.dev)
    at = 0
    for b, n in enumerate(news):
        place = torch.arange(lens[b] - n, lens[b], device=s.dev)
        p = pos[..., at:at + n] if given else place.expand(lead + (n,))
        pick = (lambda x: x[at:at + n]) if ragged else (lambda x: x[b].transpose(0, 1))
        if n:
            _close(pick(out), *_rotated(pick(q), p, rot), f"q of {b}")
        keep = place >= 0
        page, slot = s.table[b].long()[place[keep] // S], place[keep] % S
        if keep.any():
            want, size = _rotated(pick(k), p, rot)
            _close(s.k[page, :, slot], want[keep], size[keep], f"k of {b}")
            assert torch.equal(s.v[page, :, slot], pick(v)[keep])
        written[page, slot] = True
        at += n
    for now, old in zip((s.k, s.v), before):                       # every other slot as it was
        assert torch.equal(now.transpose(1, 2)[~written], old.transpose(1, 2)[~written])
    if ragged:
        assert (out[at:] == 5.0).all()
    # without queries, and without a rotation: the same entries and the plain ones
    mine = s.k.clone()
    s.k.copy_(before[0])
    assert paged_append(k, v, s.cache, s.table, s.lens, starts=starts, rotary=rot,
                        positions=pos if pos is None or ragged else pos.view(lead + (B, news[0]))) is None
    assert torch.equal(s.k, mine)
    paged_append(k, v, s.cache, s.table, s.lens, starts=starts)
    torch.cuda.synchronize()
    at = 0
    for b, n in enumerate(news):
        place = torch.arange(max(0, lens[b] - n), lens[b], device=s.dev)
        rowsb = k[at:at + n] if ragged else k[b].transpose(0, 1)
        assert torch.equal(s.k[s.table[b].long()[place // S], :, place % S], rowsb[n - len(place):])
        at += n


def test_append_in_place_queries_and_nowhere_to_put_them():
    from grammar.paged import paged_append
    from grammar.rotary import Rotary
    s = Setup([40, 40, 40], 2, 16, 64, "fp16", seed=3)
    rot = Rotary(64, device=s.dev)
    q, k, v = s.randn(3, 4, 1, 64), s.randn(3, 2, 1, 64), s.randn(3, 2, 1, 64)
    want = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot)
    got = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot, out=q)
    assert got is q and torch.equal(q, want)
    s.table[0, 2], s.table[1, 2] = -1, s.k.shape[0]                # pages that do not exist; a place behind the table
    s.lens[2] = 10_000
    before = s.k.clone(), s.v.clone()
    paged_append(s.randn(3, 2, 1, 64), s.randn(3, 2, 1, 64), s.cache, s.table, s.lens, rotary=rot)
    torch.cuda.synchronize()
    assert torch.equal(s.k, before[0]) and torch.equal(s.v, before[1])
    for starts in ([0, 3, 2, 9], [-4, -1, 7, 100], [9, 9, 9, 9]):   # starts out of order or out of the batch
        paged_append(s.randn(6, 2, 64), s.randn(6, 2, 64), s.cache, s.table, s.lens, rotary=rot,
                     starts=torch.tensor(starts, dtype=torch.int32, device=s.dev))
        torch.cuda.synchronize()


# ---- together --------------------------------------------------------------------

def test_serving_run_matches_full_attention():
    """Two conversations as a server runs them: prompts in chunks, one joining late, then decode steps, packed with a
    padded batch; every token's result against causal attention over its whole sequence in 64 bits."""
    from grammar.paged import PagedCache, paged_append, paged_attention
    from grammar.rotary import Rotary
    dev = _cuda()
    Hq, Hkv, D, S, W = 8, 2, 128, 16, 12
    rot = Rotary(D, device=dev)
    g = torch.Generator("cpu").manual_seed(6)
    total = [150, 97]
    x = [torch.randn((n, Hq + 2 * Hkv, D), generator=g).bfloat16().to(dev) for n in total]
    cache = PagedCache.empty(2 * W, Hkv, S, D, torch.bfloat16, device=dev)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    table = torch.randperm(2 * W, generator=g).int().view(2, W).to(dev)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    starts = torch.zeros(3, dtype=torch.int32, device=dev)
    rows, got = 80, [torch.empty((n, Hq, D), device=dev, dtype=torch.bfloat16) for n in total]
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
        q = paged_append(k, v, cache, table, lens, starts=starts, q=q, rotary=rot)
        o = paged_attention(q, cache, table, lens, starts=starts)
        at = 0
        for b, n in enumerate(step):
            got[b][done[b]:done[b] + n] = o[at:at + n]
            done[b] += n
            at += n
    assert done == total
    for b, n in enumerate(total):
        q, k, v = x[b].split([Hq, Hkv, Hkv], 1)
        pos = torch.arange(n, device=dev)
        # the entries as the cache holds them: rotated and rounded once
        q, k = (_rotated(t, pos, rot)[0].to(torch.bfloat16).double() for t in (q, k))
        k, v = (t.double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1).contiguous() for t in (k, v))
        sc = torch.matmul(q.transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(D)
        p = torch.softmax(sc.masked_fill(torch.ones(n, n, dtype=torch.bool, device=dev).triu(1), -math.inf), -1)
        # a rotated entry on the border of two bf16 values may round the other way: 2^-8 of some |q k| terms
        _check(got[b], torch.matmul(p, v).transpose(0, 1), torch.matmul(p, v.abs()).transpose(0, 1), f"conversation {b}",
               extra=1e-2)


def test_bound_steps_on_streams_and_in_graphs():
    """A decode loop on fixed buffers: bound once, captured, replayed as the lengths grow; two graphs, each with
    its own binding; and calls on another stream."""
    from grammar.paged import bind_paged_append, bind_paged_attention, paged_append, paged_attention
    from grammar.rotary import Rotary
    s = Setup([400, 3000], 2, 16, 128, "bf16", seed=12, width=200, spare=40)
    free = s.unused
    for b, have in ((0, 25), (1, 188)):
        for i in range(3):
            s.table[b, have + i] = free.pop()
    rot = Rotary(128, device=s.dev)
    q, k, v = s.randn(2, 8, 1, 128), s.randn(2, 2, 1, 128), s.randn(2, 2, 1, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            add, qr = bind_paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot, stream=side)
            attend, o = bind_paged_attention(qr, s.cache, s.table, s.lens, stream=side)
            add()
            attend()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                s.lens.add_(1)
                add()
                attend()
            graphs.append((graph, qr, o, add, attend))
    torch.cuda.synchronize()
    s.lens.copy_(torch.tensor([400, 3000], dtype=torch.int32))
    for i in range(8):
        graph, qr, o, *_ = graphs[i % 2]
        for t in (q, k, v):
            t.copy_(s.randn(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        s.lens_host = [401 + i, 3001 + i]
        assert s.lens.tolist() == s.lens_host
        kept = s.k.clone()
        want = paged_append(k, v, s.cache, s.table, s.lens, q=q, rotary=rot)
        assert torch.equal(want, qr) and torch.equal(kept, s.k)
        eager = paged_attention(want, s.cache, s.table, s.lens)
        assert torch.equal(eager, o)
        for b in range(2):
            ref, _, size = _attention(s, b, qr[b].transpose(0, 1))
            _check(o[b].transpose(0, 1), ref, size, f"replay {i}")
    for stream in (side, side.cuda_stream):
        side.wait_stream(torch.cuda.current_stream())
        got = paged_attention(want, s.cache, s.table, s.lens, stream=stream)
        side.synchronize()
        assert torch.equal(got, eager)


def test_scratch_goes_back_to_the_launch_stream():
    from grammar.paged import paged_attention
    s = Setup([60_000], 1, 64, 128, "fp16", seed=1)
    q = s.randn(1, 8, 40, 128)
    want = paged_attention(q, s.cache, s.table, s.lens)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()

    def free():
        return sum(b["size"] for seg in torch.cuda.memory_snapshot() if seg["stream"] == side.cuda_stream
                   for b in seg["blocks"] if b["state"] == "inactive")
    need = _needs_workspace(s, 40, 8)
    before = free()
    got = paged_attention(q, s.cache, s.table, s.lens, stream=side)
    torch.cuda.synchronize()
    assert need > 0 and free() - before >= need and torch.equal(got, want)


def test_refusals():
    from grammar import runtime as rt
    from grammar.paged import PagedCache, paged_append, paged_attention
    from grammar.rotary import Rotary
    s = Setup([20, 20], 2, 16, 64, "fp16")
    rot = Rotary(64, device=s.dev)
    q, k = s.randn(2, 4, 1, 64), s.randn(2, 2, 1, 64)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=s.dev)

    def attend(q=q, table=s.table, lens=s.lens, **kw):
        return paged_attention(q, s.cache, table, lens, **kw)

    def append(k=k, v=k, **kw):
        return paged_append(k, v, s.cache, s.table, s.lens, **kw)
    for bad in (lambda: attend(q.cpu()), lambda: attend(q.float()), lambda: attend(q[:, :3]), lambda: attend(q[..., :32]),
                lambda: attend(q[:1]), lambda: attend(table=s.table.long()), lambda: attend(lens=s.lens.long()),
                lambda: attend(lens=s.lens[:1]), lambda: attend(table=s.table[0]), lambda: attend(lens=s.lens.cpu()),
                lambda: attend(starts=starts), lambda: attend(q[:, :, 0], starts=starts[:2]), lambda: attend(q[:, :, 0]),
                lambda: attend(out=q[:, :2]), lambda: attend(workspace=torch.empty(64, dtype=torch.uint8)),
                lambda: attend(out=q[:, :1].expand(2, 4, 1, 64)), lambda: PagedCache(s.k[:1].expand(4, 2, 16, 64), s.v[:4]), lambda: attend(lse=torch.empty(2, 4, device=s.dev)),
                lambda: attend(q.transpose(1, 3).contiguous().transpose(1, 3)),
                lambda: append(k=k[:, :1]), lambda: append(v=k.bfloat16()), lambda: append(q=q), lambda: append(out=q),
                lambda: append(positions=s.lens), lambda: append(q=q, rotary=Rotary(128, device=s.dev)),
                lambda: append(q=q, rotary=rot, positions=s.lens.long()), lambda: append(q=q[:1], rotary=rot),
                lambda: append(q=q, rotary=rot, positions=torch.zeros(3, dtype=torch.int32, device=s.dev)),
                lambda: PagedCache(s.k, s.v[:1]), lambda: PagedCache(s.k.float(), s.v.float()),
                lambda: PagedCache(s.k[..., :32], s.v[..., :32]), lambda: PagedCache(s.k[:, :, :8], s.v[:, :, :8]),
                lambda: PagedCache(s.k[:, :, :12], s.v[:, :, :12]), lambda: PagedCache(s.k, s.v.bfloat16())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: attend(scale=-1.0), lambda: attend(scale=float("nan")),
                lambda: attend(torch.empty(2 * 4 * 64 + 4, device=s.dev).half()[4:].view(2, 4, 1, 64))):
        with pytest.raises(rt.GrError):
            bad()
    assert attend(q[:, :, :0]).shape == (2, 4, 0, 64)
    assert append(k=k[:, :, :0], v=k[:, :, :0]) is None
