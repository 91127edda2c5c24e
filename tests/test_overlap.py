"""Outputs that share memory with other arrays of a call are refused: the check
itself against sets of elements, and the entry points' refusals (no GPU; the
addresses are never followed)."""
import ctypes
import random

import pytest
import torch


def _elements(t):
    """Places of t's elements, in its element's size from address 0."""
    at = torch.full(t.shape, t.data_ptr() // t.element_size(), dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at = at + (torch.arange(n) * s).view([-1 if i == d else 1 for i in range(t.dim())])
    return set(at.flatten().tolist())


def _overlap(a, b):
    from grammar import runtime as rt
    four = ctypes.c_longlong * 4
    return rt.lib().gr_selftest_overlap(a.data_ptr(), four(*a.shape), four(*a.stride()),
                                        b.data_ptr(), four(*b.shape), four(*b.stride()), a.element_size())


def _check(a, b):
    want = bool(_elements(a) & _elements(b))
    assert _overlap(a, b) == want == _overlap(b, a), (a.shape, a.stride(), b.shape, b.stride(), b.storage_offset())
    return want


def test_slices_of_one_projection():
    rows = torch.zeros(2, 5, 14, 16)
    q, k, v = (rows[:, :, i:j].transpose(1, 2) for i, j in ((0, 8), (8, 10), (10, 14)))
    assert not _check(q, k) and not _check(k, v) and not _check(q, v) and _check(q, q)
    assert _check(q, rows[:, :, 7:9].transpose(1, 2)) and _check(q[:, :, 1:], q[:, :, :-1])
    assert not _check(q[:, :, ::2], q[:, :, 1::2]) and not _check(q[..., :8], q[..., 8:])
    assert not _check(q, torch.zeros_like(q)) and not _check(q[:, :, :0], q)
    assert _check(rows[:, :, :8].transpose(1, 2), rows.view(-1)[:2 * 8 * 5 * 16].view(2, 8, 5, 16))
    assert _check(q[:1, :1, :1], q.expand(2, 8, 5, 16)) and _check(q[:, :1].expand(2, 8, 5, 16), q[:, :1])
    long = torch.zeros(1).expand(4096, 4096, 4096, 4096)                # strides of 0 are no search
    assert _overlap(long, long)


@pytest.mark.parametrize("seed", range(300))
def test_random_views(seed):
    rng = random.Random(seed)
    base = torch.zeros(4000)

    def view():
        shape = [rng.choice((1, 2, 3, 5)) for _ in range(3)] + [rng.choice((1, 4, 8))]
        st, step = [0] * 4, rng.choice((1, 1, 2))
        for d in [3] + rng.sample(range(3), 3):
            st[d] = step
            step = step * shape[d] + rng.choice((0, 0, 1, 4, 7))
            step *= rng.choice((1, 1, 2))
        size = sum((n - 1) * s for n, s in zip(shape, st)) + 1
        return base.as_strided(shape, st, rng.randrange(0, 4000 - size)) if size < 4000 else base[:8].view(1, 1, 1, 8)
    a, b = view(), view()
    _check(a, b)
    # and close together, where both answers are frequent
    off = min(a.storage_offset() + rng.randrange(0, 12), 4000 - sum((n - 1) * s for n, s in zip(b.shape, b.stride())) - 1)
    _check(a, base.as_strided(b.shape, b.stride(), off))


AT = 1 << 30


def _rotary(q_out, k_out, *, q=AT, k=AT + (1 << 24), N=9, st=(9 * 512, 512, 64), q_out_st=None, k_heads=2):
    """gr_rotary of 8 query heads of 64 in fp16: its status and message."""
    from grammar import runtime as rt
    spec = rt.RotarySpec(AT, AT, 32, 1, 64, 0)
    s = rt._ll3(*st)
    rc = rt.lib().gr_rotary(ctypes.addressof(spec), q, q_out, 8, s, rt._ll3(*(q_out_st or st)), k, k_out, k_heads, s, s,
                            rt.GR_F16, 2, N, AT, rt._ll3(0, 0, 1), 0, None)
    return rc, rt.last_error()


def test_rotary_refuses_outputs_over_inputs():
    from grammar import runtime as rt
    far, k = AT + (1 << 26), AT + (1 << 24)
    for case, name in (((k, far), "q_out"), ((far, AT), "k_out"), ((k, AT), "q_out"),       # the other's input
                       ((far, far), "q_out"), ((far, far + 2 * 64 * 2), "q_out"),           # two outputs in one place
                       ((AT + 2 * 64 * 4, far), "q_out"), ((far, k + 16 * 2), "k_out"),     # a part of its own
                       ((AT - 2 * 512, far), "q_out")):                                     # a token behind
        rc, msg = _rotary(*case)
        assert rc == rt.GR_E_ARG and name in msg and "shares memory" in msg, (case, rc, msg)
    rc, msg = _rotary(AT, far, q_out_st=(9 * 512, 64, 9 * 64))                              # its own, transposed
    assert rc == rt.GR_E_ARG and "q_out" in msg and "shares memory" in msg
    rc, msg = _rotary(far, None, k=AT, k_heads=2)
    assert rc == rt.GR_E_ARG and "null" in msg


def test_paged_calls_refuse_outputs_over_other_arrays():
    from grammar import runtime as rt
    k_pages, v_pages, q, k, v, table, far = (AT + (i << 26) for i in range(7))
    strides = (4096, 1024, 64)
    cache = rt.PagedCacheDesc(k_pages, v_pages, rt._ll3(*strides), rt._ll3(*strides), rt.GR_BF16, 8, 4, 16, 64)
    for starts in (None, table):
        batch = rt.PagedBatch(table, 8, table, starts, 2, 3, 8, 0, 0)
        spec = rt.RotarySpec(table, table, 32, 1, 64, 0)
        p, qs, ks = ctypes.addressof, rt._ll3(3 * 512, 512, 64), rt._ll3(3 * 256, 256, 64)
        for out in (k_pages, v_pages, v_pages + 2 * 8 * 4096 - 128, q + 128, q - 128):
            rc = rt.lib().gr_paged_attn(p(cache), p(batch), q, out, None, 8, qs, qs, 1, 0.125, None, 0, None)
            assert rc == rt.GR_E_ARG and "shares memory" in rt.last_error(), (out, rt.last_error())
        for out in (k, v, k + 2 * 256 - 16, k_pages, v_pages, q + 128):
            rc = rt.lib().gr_paged_append(p(cache), p(batch), p(spec), q, out, 8, qs, qs, k, v, ks, ks, None, None, None)
            assert rc == rt.GR_E_ARG and "shares memory" in rt.last_error(), (out, rt.last_error())
