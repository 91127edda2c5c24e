"""The entry points of normed heads and of a quantised paged cache: what they refuse
before anything is launched (no GPU; the addresses are never followed)."""
import ctypes
import re

import pytest

from test_paged_cpu import BAD_BATCH, BAD_CACHE, _parts


def _scales(d, rt):
    return rt.PagedScales(d + (1 << 16), rt._ll3(128, 32, 16))


def _calls(rt, d, cache, scales, batch, spec, norm=None):
    """Every entry point over a quantised cache."""
    p, s = ctypes.addressof, rt._ll3(512, 64, 64)
    L = rt.lib()
    c, sc, b = p(cache), p(scales) if scales else None, p(batch)
    far = d + (1 << 24)
    keep = (cache, scales, batch, spec, norm)                               # what the addresses are of
    return (lambda keep=keep: L.gr_paged_append_with(c, sc, b, p(spec), p(norm) if norm else None, None, None, 0, None, None, far, far, s, s,
                                           None, None, None),
            lambda keep=keep: L.gr_paged_attn_scaled(c, sc, b, far, far, None, 8, s, s, 1, 0.125, None, 0, None),
            lambda keep=keep: L.gr_paged_read(c, sc, b, far, far + (1 << 24), s, s, None))


@pytest.mark.parametrize("what,field,value,msg", [("cache", *c) for c in BAD_CACHE] + [("batch", *c) for c in BAD_BATCH])
def test_bad_caches_and_batches_are_refused(what, field, value, msg):
    rt, d, cache, batch, spec = _parts()
    scales = _scales(d, rt)
    setattr(cache if what == "cache" else batch, field, value)
    for call in _calls(rt, d, cache, scales, batch, spec):
        assert call() == rt.GR_E_ARG
        assert re.search(msg, rt.last_error()), rt.last_error()
    p = ctypes.addressof
    assert rt.lib().gr_paged_attn_scaled_workspace(p(cache), p(scales), p(batch), 8) == 0


def test_bad_scales_are_refused():
    rt, d, cache, batch, spec = _parts()
    scales = _scales(d, rt)
    scales.scales = None
    for call in _calls(rt, d, cache, scales, batch, spec):
        assert call() == rt.GR_E_ARG and "null" in rt.last_error()
    for i in range(3):
        scales = _scales(d, rt)
        for bad in (-16, 8):
            scales.strides[i] = bad
            for call in _calls(rt, d, cache, scales, batch, spec):
                assert call() == rt.GR_E_ARG and "strides" in rt.last_error()
    scales = _scales(d, rt)
    scales.scales += 8
    for call in _calls(rt, d, cache, scales, batch, spec):
        assert call() == rt.GR_E_ARG and "aligned" in rt.last_error()
    scales = _scales(d, rt)
    for i, (s, keep) in enumerate(((4104, 4096), (1032, 1024), (72, 64))):      # multiples of 8, not of 16
        for strides in (cache.k_strides, cache.v_strides):
            strides[i] = s
            for call in _calls(rt, d, cache, scales, batch, spec):
                assert call() == rt.GR_E_ARG and "16" in rt.last_error()
            strides[i] = keep
    p, s = ctypes.addressof, rt._ll3(512, 64, 64)
    assert rt.lib().gr_paged_attn_scaled(p(cache), None, p(batch), d, d, None, 8, s, s, 1, 0.125, None, 0, None) == rt.GR_E_ARG
    assert rt.lib().gr_paged_attn_scaled_workspace(p(cache), None, p(batch), 8) == 0


@pytest.mark.parametrize("field,value,msg", [("q_weight", (1 << 20) + 8, "aligned"), ("k_weight", (1 << 20) + 4, "aligned"),
                                             ("dtype", 1, "type"), ("dtype", 7, "type"), ("eps", -1.0, "eps"),
                                             ("eps", float("nan"), "eps"), ("eps", float("inf"), "eps")])
def test_bad_norms_are_refused(field, value, msg):
    rt, d, cache, batch, spec = _parts()
    norm = rt.HeadNormSpec(d, d, rt.GR_BF16, 1e-6)
    setattr(norm, field, value)
    call = _calls(rt, d, cache, _scales(d, rt), batch, spec, norm)[0]
    assert call() == rt.GR_E_ARG and msg in rt.last_error(), rt.last_error()
    p, s = ctypes.addressof, rt._ll3(512, 64, 64)
    L, far = rt.lib(), d + (1 << 24)
    assert L.gr_norm_rotary(p(spec), p(norm), d, far, 1, s, s, None, None, 0, None, None, rt.GR_BF16, 1, 1, d, s, None) == rt.GR_E_ARG
    assert msg in rt.last_error()
    assert L.gr_norm_rotary_bwd(p(spec), p(norm), d, d, far, 1, s, s, s, None, None, None, 0, None, None, None, rt.GR_BF16, 1, 1, d, s,
                                None, None, None, 0, None) == rt.GR_E_ARG
    assert msg in rt.last_error()


def test_bad_norm_calls_are_refused():
    rt, d, cache, batch, spec = _parts()
    p, s, L = ctypes.addressof, rt._ll3(512, 64, 64), rt.lib()
    norm = rt.HeadNormSpec(d, d, rt.GR_BF16, 1e-6)
    far = [d + (i << 24) for i in range(1, 8)]
    n, r = p(norm), p(spec)
    bf = rt.GR_BF16
    for args, msg in (((r, None, d, far[0], 1, s, s, None, None, 0, None, None, bf, 1, 1, d, s, None), "null"),
                      ((r, n, None, far[0], 1, s, s, None, None, 0, None, None, bf, 1, 1, d, s, None), "null"),
                      ((r, n, d, far[0], 1, s, s, None, None, 0, None, None, 5, 1, 1, d, s, None), "dtype"),
                      ((r, n, d, far[0], 0, s, s, None, None, 0, None, None, bf, 1, 1, d, s, None), "head"),
                      ((r, n, d, far[0], 1, s, s, d, far[0], 1, s, s, bf, 1, 1, d, s, None), "memory"),
                      ((r, n, far[1], d, 1, s, s, None, None, 0, None, None, bf, 1, 1, far[2], s, None), "weights"),
                      ((r, n, far[1], far[2], 1, s, s, far[3], d + 64, 1, s, s, bf, 1, 1, far[4], s, None), "weights"),
                      ((r, n, d, far[0], 1, s, s, None, None, 0, None, None, bf, 1 << 16, 1 << 16, d, s, None), "positive")):
        assert L.gr_norm_rotary(*args) == rt.GR_E_ARG and msg in rt.last_error(), rt.last_error()

    at_q = rt.HeadNormSpec(far[3], None, rt.GR_F32, 1e-6)
    assert L.gr_paged_append_with(p(cache), None, p(batch), r, p(at_q), far[5], far[3], 8, s, s, far[6], far[6], s, s, None, None,
                                  None) == rt.GR_E_ARG
    assert "weights" in rt.last_error(), rt.last_error()

    def bwd(q=d, g=far[0], dq=far[1], k=far[2], gk=far[3], dk=far[4], wq=far[5], wk=far[6], ws=d + (9 << 24), size=1 << 20, N=1):
        return L.gr_norm_rotary_bwd(r, n, q, g, dq, 1, s, s, s, k, gk, dk, 1, s, s, s, bf, 1, N, d, s, wq, wk, ws, size, None)
    for kw, msg in ((dict(q=None), "null"), (dict(g=None), "null"), (dict(gk=None), "null"), (dict(dk=None), "null"), (dict(dq=far[3]), "memory"),
                    (dict(dq=far[2]), "memory"), (dict(dq=far[4]), "memory"), (dict(q=far[6], wk=None, dq=d + 96), "weights"), (dict(q=far[6], wk=None, dk=d), "weights"), (dict(wq=far[1]), "memory"), (dict(wk=far[4] + 64), "memory"),
                    (dict(wq=far[6]), "memory"), (dict(wq=far[5] + 2), "aligned"), (dict(ws=None), "workspace"), (dict(size=100), "workspace"),
                    (dict(ws=d + 4), "workspace"), (dict(N=0), "positive"), (dict(dq=d + 16, N=9), "memory")):
        assert bwd(**kw) == rt.GR_E_ARG and msg in rt.last_error(), (kw, rt.last_error())


def test_norm_workspace_sizes():
    rt, *_ = _parts()
    size = rt.lib().gr_norm_rotary_bwd_workspace
    assert size(8, 2, 64, 1, 1) == 2 * 64 * 4                   # one workgroup
    many = size(32, 8, 128, 2, 4096)
    assert many % (2 * 128 * 4) == 0 and 1 << 18 <= many <= 1 << 23
    for bad in ((0, 2, 64), (8, -1, 64), (8, 2, 72), (8, 2, 512), (8, 2, 0)):
        assert size(*bad, 1, 1) == 0
    assert size(8, 2, 64, 0, 1) == 0


def test_no_rows_are_no_work():
    rt, d, cache, batch, spec = _parts()
    batch.rows = 0
    for call in _calls(rt, d, cache, _scales(d, rt), batch, spec):
        assert call() == 0


def test_cpu_tensors_are_refused():
    import torch
    from grammar.norm import HeadNorm, norm_rotary
    from grammar.paged import QuantizedPagedCache
    from grammar.rotary import Rotary
    with pytest.raises(ValueError, match="GPU"):
        QuantizedPagedCache.empty(4, 2, 16, 64, torch.float16, device="cpu")
    rot = Rotary(64, device="cpu")
    with pytest.raises(ValueError, match="CPU"):
        norm_rotary(torch.zeros(1, 1, 3, 64), None, torch.zeros(3, dtype=torch.int32), rot, HeadNorm())
