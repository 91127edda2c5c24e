"""Paged attention and appending at the edges of what they promise."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_paged_gpu import Setup, _attention, _check, _check_lse  # noqa: E402


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("w", [23.4, 24.6, 25.05, 26.5])
@pytest.mark.parametrize("n,G,D,alone", [(1, 4, 64, False), (1, 4, 128, True), (5, 7, 64, True), (200, 2, 64, True),
                                         (200, 2, 128, False), (4100, 8, 64, True), (4100, 8, 128, True)])
def test_many_small_weights_add_up(dtype, w, n, G, D, alone):
    """One key of weight 1 and value 1, then N of about 2^-w and value -1: a row that sees M' = N p of the latter is
    (1 - M') / (1 + M'), its log-sum-exp log(1 + M'). In tiles of all sizes, a workgroup a tile and shared out."""
    from grammar.paged import paged_attention
    N = 50_001
    print(f"[case] small weights {dtype} w {w} n{n} G{G} D{D} alone={alone}", flush=True)
    s = Setup([N], 1, 64, D, dtype)
    s.k.zero_()
    s.k[..., 0] = -w * math.log(2)
    s.v.fill_(-1.0)
    first = int(s.table[0, 0])
    x = float(s.k[first, 0, 1, 0])                               # the score as it is stored
    s.k[first, 0, 0] = 0
    s.v[first, 0, 0] = 1
    q = torch.zeros(1, G, n, D, dtype=s.dtype, device=s.dev)
    q[..., 0] = 1
    lse = torch.empty(1, n, G, device=s.dev)
    got = paged_attention(q, s.cache, s.table, s.lens, scale=1.0, lse=lse,
                          workspace=torch.empty(0, dtype=torch.uint8, device=s.dev) if alone else None)
    m = (N - n + torch.arange(n, dtype=torch.float64, device=s.dev)) * math.exp(x)
    want = ((1 - m) / (1 + m))[None, None, :, None]
    # p rounds by half a step of itself and is off by its exponent's rounding (2^-24 of 40) and 2^-22, which is what M'
    # and log(1 + M') are off by, and half of what (1 - M') / (1 + M') is; in fp16 all keys far below the base lose 2^-14
    # of it at most. fp32 sums: a rounding for each 4 keys at least, 2^-24 of a sum of about 1. The result rounds once.
    u = torch.finfo(s.dtype).eps / 2
    sums = N / 4 * 2.0 ** -24
    off = float(m.max()) * (u + 40 * 2.0 ** -24 + 2.0 ** -22) + (2.0 ** -14 if dtype == "fp16" else 0)
    assert ((got.double() - want).abs() <= 2 * off + sums + u * want.abs()).all(), \
        float((got.double() - want).abs().max())
    assert ((lse.double() - torch.log1p(m)[None, :, None]).abs() <= off + sums + 2.0 ** -22).all(), \
        float((lse.double() - torch.log1p(m)[None, :, None]).abs().max())


@pytest.mark.parametrize("starts,rows_of", [([0, 3, 9], {0: (0, 3)}), ([-2, 3, 6], {1: (3, 6)}), ([-1, 7, 8], {}),
                                            ([0, 0, 7], {})])
def test_sequences_out_of_the_batch_append_nothing(starts, rows_of):
    """A sequence whose rows are not all in the batch has no new tokens, to appends as to attention."""
    from grammar.paged import paged_append, paged_attention
    from grammar.rotary import Rotary
    s = Setup([40, 50], 2, 16, 64, "fp16", seed=5)
    rot = Rotary(64, device=s.dev)
    print(f"[case] starts {starts}", flush=True)
    q, k, v = s.randn(6, 4, 64), s.randn(6, 2, 64), s.randn(6, 2, 64)
    at = torch.tensor(starts, dtype=torch.int32, device=s.dev)
    before = s.k.clone(), s.v.clone()
    out, o = torch.full_like(q, 5.0), torch.full_like(q, 5.0)
    paged_append(k, v, s.cache, s.table, s.lens, starts=at, q=q, rotary=rot, out=out)
    paged_attention(q, s.cache, s.table, s.lens, starts=at, out=o)
    written = torch.zeros(s.k.shape[0], s.S, dtype=torch.bool, device=s.dev)
    rows = torch.zeros(6, dtype=torch.bool, device=s.dev)
    for b, (r0, r1) in rows_of.items():
        place = torch.arange(s.lens_host[b] - (r1 - r0), s.lens_host[b], device=s.dev)
        page, slot = s.table[b].long()[place // s.S], place % s.S
        written[page, slot] = True
        rows[r0:r1] = True
        assert torch.equal(s.v[page, :, slot], v[r0:r1])
    for now, old in zip((s.k, s.v), before):
        assert torch.equal(now.transpose(1, 2)[~written], old.transpose(1, 2)[~written])
    for x in (out, o):
        assert (x[~rows] == 5.0).all() and (x[rows] != 5.0).any(-1).all()


@pytest.mark.parametrize("D,hint", [(64, 1), (64, 0), (128, 1), (128, 0)])
def test_overlapping_starts_stay_in_bounds(D, hint):
    """Every second sequence claims all of the batch's rows: more tiles than the grid has, and more blocks of keys than
    32 bits count. The rows of no other call are touched, and every row gets the result that any of them would give."""
    from grammar.paged import paged_attention
    B, rows, W = 512, 16_384, 65_536
    print(f"[case] overlapping starts D{D} hint {hint}", flush=True)
    s = Setup([16], 2, 16, D, "bf16")
    table = torch.full((1, W), -1, dtype=torch.int32, device=s.dev).expand(B, W)
    lens = torch.full((B,), W * 16, dtype=torch.int32, device=s.dev)
    starts = torch.tensor([0, rows] * (B // 2) + [0], dtype=torch.int32, device=s.dev)
    q = s.randn(rows, 2, D)
    for ws in (None, torch.empty(0, dtype=torch.uint8, device=s.dev)):
        out = torch.full((rows + 64, 2, D), 5.0, dtype=s.dtype, device=s.dev)
        paged_attention(q, s.cache, table, lens, starts=starts, max_new=hint, out=out[32:-32], workspace=ws)
        torch.cuda.synchronize()
        assert not out[32:-32].any() and (out[:32] == 5.0).all() and (out[-32:] == 5.0).all()


def test_caches_and_rotations_can_be_copied_and_pickled():
    import copy
    import pickle
    from grammar.paged import PagedCache, paged_append, paged_attention
    from grammar.rotary import Rotary
    s = Setup([40, 50], 2, 16, 64, "fp16", seed=6)
    rot = Rotary(64, device=s.dev)
    both = torch.stack((s.k, s.v), 1)                            # keys and values in one tensor
    q, k, v = s.randn(2, 4, 1, 64), s.randn(2, 2, 1, 64), s.randn(2, 2, 1, 64)
    for cache in (s.cache, PagedCache(both[:, 0], both[:, 1])):
        for make in (copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
            c, r = make((cache, rot))
            assert type(c) is PagedCache and c.desc.k == c.k.data_ptr() != cache.k.data_ptr()
            assert torch.equal(c.k, cache.k) and torch.equal(c.v, cache.v) and c.k.stride() == cache.k.stride()
            old = cache.k.clone()
            qr = paged_append(k, v, c, s.table, s.lens, q=q, rotary=r)
            got = paged_attention(qr, c, s.table, s.lens)
            assert torch.equal(cache.k, old)                     # the copy's pages are its own
            there = make(cache)
            assert torch.equal(paged_append(k, v, there, s.table, s.lens, q=q, rotary=rot), qr)
            assert torch.equal(paged_attention(qr, there, s.table, s.lens), got)
        shared = copy.copy(cache)
        assert shared.k is cache.k and shared.ref != cache.ref


def test_outputs_share_memory_with_their_own_input_only():
    from grammar import runtime as rt
    from grammar.paged import paged_append, paged_attention
    from grammar.rotary import Rotary, rotary_fwd
    s = Setup([40, 50, 300], 2, 16, 64, "fp16", seed=7)
    rot = Rotary(64, device=s.dev)
    n, starts = 9, torch.tensor([0, 9, 18, 27], dtype=torch.int32, device=s.dev)
    rows = s.randn(27, 14, 64)                                   # a projection's rows: 8 q, 2 k, 2 v heads and 2 more
    q, k, v = rows[:, :8], rows[:, 8:10], rows[:, 10:12]
    args = (s.cache, s.table, s.lens)
    for bad in (lambda: paged_append(k, v, *args, starts=starts, q=q, rotary=rot, out=rows[:, 4:12]),
                lambda: paged_append(k, v, *args, starts=starts, q=k, rotary=rot, out=v),
                lambda: paged_append(k, v, *args, starts=starts, q=q, rotary=rot, out=rows.view(-1)[:27 * 512].view(27, 8, 64)),
                lambda: paged_attention(q, *args, starts=starts, out=rows[:, 6:14]),
                lambda: paged_attention(q, *args, starts=starts, out=s.k.view(-1)[:27 * 512].view(27, 8, 64)),
                lambda: rotary_fwd(q[None].transpose(1, 2), k[None].transpose(1, 2), starts[:1].expand(27), rot,
                                   out=rows[None, :, 2:10].transpose(1, 2))):
        before = rows.clone(), s.k.clone()
        with pytest.raises(rt.GrError, match="shares memory"):
            bad()
        assert torch.equal(rows, before[0]) and torch.equal(s.k, before[1])
    # in place, and into other heads of the same rows
    want = paged_append(k, v, *args, starts=starts, q=q, rotary=rot)
    wide = s.randn(27, 24, 64)
    wide[:, :14] = rows
    got = paged_append(wide[:, 8:10], wide[:, 10:12], *args, starts=starts, q=wide[:, :8], rotary=rot, out=wide[:, 16:])
    assert torch.equal(got, want) and torch.equal(wide[:, :14], rows)
    paged_append(k, v, *args, starts=starts, q=q, rotary=rot, out=q)
    assert torch.equal(q, want)
    # attention in place: in tiles of 32, 64 and 128 rows, a workgroup a tile and shared out
    for m, lens, width in ((1, [40, 50, 3000], None), (9, [40, 50, 300], None), (150, [150, 500, 4000], None),
                           (1, [40, 50, 3000], 2048), (150, [150, 500, 4000], 2048)):
        t = Setup(lens, 2, 16, 64, "fp16", seed=m, width=width)
        x = t.randn(3, 8, m, 64)
        o = paged_attention(x, t.cache, t.table, t.lens)
        assert paged_attention(x, t.cache, t.table, t.lens, out=x) is x and torch.equal(x, o)


HINTS = [dict(max_new=1, max_len=1), dict(max_new=1), dict(max_len=1), dict(max_new=20, max_len=700),
         dict(max_new=2 ** 31 - 1, max_len=2 ** 31 - 1), dict(max_new=-5, max_len=-5)]


@pytest.mark.parametrize("hints", HINTS, ids=lambda h: "-".join(f"{k[4:]}{v}" for k, v in h.items()))
@pytest.mark.parametrize("dtype,D,G,Hkv", [("bf16", 128, 4, 2), ("fp16", 64, 1, 4)])
@pytest.mark.parametrize("width", [None, 2048], ids=["fit", "roomy"])
def test_hints_that_do_not_hold(hints, dtype, D, G, Hkv, width):
    """max_new and max_len only choose how the work is shared out: a bound loop outgrows them. A packed batch of chunks
    and single tokens, decode steps over long contexts and a chunk of its own, with hints too small and too large."""
    from grammar.paged import paged_append, paged_attention
    print(f"[case] hints {hints} {dtype} D{D} width {width}", flush=True)
    for news, lens, ragged in (([1, 0, 150, 1, 7, 301, 1], [40, 99, 150, 700, 7, 900, 0], True),
                               ([1, 1, 1], [20_011, 3, 5000], False), ([200], [5000], False)):
        s = Setup(lens, Hkv, 16, D, dtype, seed=D, width=width)
        T, B, Hq = sum(news) + 3 * ragged, len(news), G * Hkv
        q = s.randn(T, Hq, D) if ragged else s.randn(B, Hq, news[0], D)
        starts = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device=s.dev) if ragged else None
        out, lse = torch.full_like(q, 5.0), torch.full((T, Hq) if ragged else (B, news[0], Hq), 7.0, device=s.dev)
        paged_attention(q, s.cache, s.table, s.lens, starts=starts, out=out, lse=lse, **hints)
        for b, n in enumerate(news):
            pick = (lambda x: x[sum(news[:b]):sum(news[:b + 1])]) if ragged else (lambda x: x[b].transpose(0, 1))
            o, ls, size = _attention(s, b, pick(q))
            _check(pick(out), o, size, f"{n} of {lens[b]} keys")
            _check_lse(pick(lse) if ragged else lse[b], ls, s.dtype, f"lse of {b}")
        if ragged:
            assert (out[sum(news):] == 5.0).all() and (lse[sum(news):] == 7.0).all()
            k, v = s.randn(T, Hkv, D), s.randn(T, Hkv, D)
            paged_append(k, v, s.cache, s.table, s.lens, starts=starts, max_new=hints.get("max_new", 0))
            page, slot = int(s.table[5, 899 // 16]), 899 % 16
            assert torch.equal(s.k[page, :, slot], k[459]) and torch.equal(s.v[page, :, slot], v[459])


@pytest.mark.parametrize("pad,off", [(128, 8), (128, 32), (136, 0), (192, 0)])
def test_destinations_off_a_line(pad, off):
    """Results in rows that begin off a 128-byte line, and pages with padded slots: bit for bit the packed ones, and
    nothing behind a row is written."""
    from grammar.paged import PagedCache, paged_append
    from grammar.rotary import Rotary, rotary_fwd
    s = Setup([700, 900], 8, 16, 128, "bf16", seed=8)
    rot = Rotary(128, device=s.dev)
    print(f"[case] rows of {pad}, {off} off", flush=True)

    def rows(*shape):
        n = math.prod(shape)
        x = torch.full((n * pad + 64,), 5.0, dtype=s.dtype, device=s.dev)
        whole = x[off:off + n * pad].view(*shape, pad)
        return whole[..., :128], lambda: (whole[..., 128:] == 5.0).all() and (x[:off] == 5.0).all() and (x[off + n * pad:] == 5.0).all()
    q, k = s.randn(1, 32, 600, 128), s.randn(1, 8, 600, 128)
    pos = torch.arange(600, dtype=torch.int32, device=s.dev)
    (o, o_kept), (ko, ko_kept) = rows(1, 32, 600), rows(1, 8, 600)
    want = rotary_fwd(q, k, pos, rot)
    rotary_fwd(q, k, pos, rot, out=o, k_out=ko)
    assert torch.equal(o, want[0]) and torch.equal(ko, want[1]) and o_kept() and ko_kept()
    q, k = s.randn(2, 32, 600, 128), s.randn(2, 8, 600, 128)
    pages = [rows(s.k.shape[0], 8, 16) for _ in range(2)]
    for (p, _), x in zip(pages, (s.k, s.v)):
        p.copy_(x)
    cache, (o, o_kept) = PagedCache(pages[0][0], pages[1][0]), rows(2, 32, 600)
    want = paged_append(k, k, s.cache, s.table, s.lens, q=q, rotary=rot)
    paged_append(k, k, cache, s.table, s.lens, q=q, rotary=rot, out=o)
    assert torch.equal(o, want) and torch.equal(cache.k, s.k) and torch.equal(cache.v, s.v)
    assert o_kept() and pages[0][1]() and pages[1][1]()


def test_calls_of_two_threads_at_once():
    """Two host threads, each with a stream and a cache of its own and calls whose work is shared out, in flight at once."""
    import threading
    from grammar.paged import paged_append, paged_attention
    from grammar.rotary import Rotary
    rot = Rotary(128, device=torch.device("cuda:0"))
    sides = [torch.cuda.Stream() for _ in range(2)]
    cases = []
    for i in range(2):
        s = Setup([4000 + 900 * i, 70, 2500], 2, 16, 128, "bf16", seed=20 + i, width=400)
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
