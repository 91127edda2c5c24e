"""The entry points over a paged cache and the position rotation: what they
refuse before anything is launched, and the tables a Rotary holds (no GPU)."""
import ctypes
import math

import pytest
import torch


def _parts():
    from grammar import runtime as rt
    dummy = 1 << 20                                     # an aligned address that is never followed
    cache = rt.PagedCacheDesc(dummy, dummy, rt._ll3(4096, 1024, 64), rt._ll3(4096, 1024, 64), rt.GR_BF16, 8, 4, 16, 64)
    batch = rt.PagedBatch(dummy, 8, dummy, None, 2, 1, 8, 0, 0)
    spec = rt.RotarySpec(dummy, dummy, 32, 1, 64, 0)
    return rt, dummy, cache, batch, spec


def _attn(cache, batch, **kw):
    rt, d, *_ = _parts()
    a = dict(q=d, o=d, lse=None, Hq=8, qs=rt._ll3(512, 64, 64), os=rt._ll3(512, 64, 64), scale=0.125, ws=None, size=0)
    a.update(kw)
    p = ctypes.addressof
    return rt.lib().gr_paged_attn(p(cache) if cache else None, p(batch) if batch else None, a["q"], a["o"], a["lse"],
                                  a["Hq"], a["qs"], a["os"], 1, a["scale"], a["ws"], a["size"], None)


BAD_CACHE = [("k", 0, "null"), ("v", 0, "null"), ("k", (1 << 20) + 8, "aligned"), ("dtype", 0, "dtype"), ("dtype", 7, "dtype"),
             ("head_dim", 96, "head dim"), ("pages", 0, "pages"), ("heads", 0, "heads"), ("page_size", 8, "page size"),
             ("page_size", 48, "page size"), ("page_size", 0, "page size"), ("page_size", -16, "page size")]
BAD_BATCH = [("table", 0, "null"), ("lens", 0, "null"), ("B", 0, "positive"), ("rows", -1, "positive"),
             ("width", 0, "positive"), ("width", 1 << 27, "2\\^30"), ("rows", (1 << 31) - 1, "too many")]


@pytest.mark.parametrize("what,field,value,msg", [("cache", *c) for c in BAD_CACHE] + [("batch", *c) for c in BAD_BATCH])
def test_bad_caches_and_batches_are_refused(what, field, value, msg):
    rt, d, cache, batch, spec = _parts()
    setattr(cache if what == "cache" else batch, field, value)
    assert _attn(cache, batch) == rt.GR_E_ARG
    import re
    assert re.search(msg, rt.last_error()), rt.last_error()
    assert rt.lib().gr_paged_attn_workspace(ctypes.addressof(cache), ctypes.addressof(batch), 8) == 0
    p, s = ctypes.addressof, rt._ll3(256, 64, 64)
    rc = rt.lib().gr_paged_append(p(cache), p(batch), p(spec), None, None, 0, None, None, d, d, s, s, None, None, None)
    assert rc == rt.GR_E_ARG


def test_strides_of_the_cache_are_checked():
    rt, d, cache, batch, spec = _parts()
    for i, s in ((0, 4095), (1, -8), (2, 1 << 27)):
        cache.k_strides[i], keep = s, cache.k_strides[i]
        assert _attn(cache, batch) == rt.GR_E_ARG and "strides" in rt.last_error()
        cache.k_strides[i] = keep


@pytest.mark.parametrize("kw,msg", [
    (dict(q=None), "null"), (dict(o=None), "null"), (dict(q=(1 << 20) + 2), "aligned"), (dict(lse=(1 << 20) + 2), "lse"),
    (dict(Hq=6), "multiple"), (dict(Hq=0), "multiple"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(ws=(1 << 20) + 4, size=1 << 20), "aligned")])
def test_bad_attention_arguments_are_refused(kw, msg):
    rt, d, cache, batch, spec = _parts()
    assert _attn(cache, batch, **kw) == rt.GR_E_ARG
    assert msg in rt.last_error()


def test_null_structures_are_refused():
    rt, d, cache, batch, spec = _parts()
    assert _attn(None, batch) == rt.GR_E_ARG and _attn(cache, None) == rt.GR_E_ARG
    assert rt.lib().gr_rotary(None, d, d, 1, None, None, None, None, 0, None, None, 1, 1, 1, d, None, 0, None) == rt.GR_E_ARG


def test_no_new_tokens_is_no_work():
    rt, d, cache, batch, spec = _parts()
    batch.rows = 0
    assert _attn(cache, batch, q=None, o=None) == 0
    assert rt.lib().gr_paged_attn_workspace(ctypes.addressof(cache), ctypes.addressof(batch), 8) == 0


@pytest.mark.parametrize("field,value,msg", [
    ("turns", 0, "turns"), ("turns", (1 << 20) + 4, "turns"), ("pairs", 12, "pairs"), ("pairs", 0, "pairs"),
    ("pairs", 40, "pairs"), ("naxes", 0, "axes"), ("naxes", 9, "axes"), ("head_dim", 72, "head dim"),
    ("head_dim", 512, "head dim")])
def test_bad_rotations_are_refused(field, value, msg):
    rt, d, cache, batch, spec = _parts()
    setattr(spec, field, value)
    s = rt._ll3(256, 64, 64)
    rc = rt.lib().gr_rotary(ctypes.addressof(spec), d, d, 1, s, s, None, None, 0, None, None, rt.GR_BF16, 1, 1, d, s, 0, None)
    assert rc == rt.GR_E_ARG and msg in rt.last_error()


def test_bad_rotary_calls_are_refused():
    rt, d, cache, batch, spec = _parts()
    s, p = rt._ll3(256, 64, 64), ctypes.addressof(spec)
    call = rt.lib().gr_rotary
    for args, msg in (((p, None, d, 1, s, s, None, None, 0, None, None, 2, 1, 1, d, s, 0, None), "null"),
                      ((p, d, d, 0, s, s, None, None, 0, None, None, 2, 1, 1, d, s, 0, None), "head"),
                      ((p, d, d, 1, s, s, d, None, 1, s, s, 2, 1, 1, d, s, 0, None), "null"),
                      ((p, d, d, 1, rt._ll3(4, 64, 64), s, None, None, 0, None, None, 2, 1, 1, d, s, 0, None), "strides"),
                      ((p, d, d, 1, s, s, None, None, 0, None, None, 3, 1, 1, d, s, 0, None), "dtype"),
                      ((p, d, d, 1, s, s, None, None, 0, None, None, 2, 1 << 16, 1 << 16, d, s, 0, None), "positive"),
                      ((p, d, d, 1, s, s, None, None, 0, None, None, 2, 0, 1, d, s, 0, None), "positive"),
                      ((p, d, d, 1, s, s, None, None, 0, None, None, 2, 1, 1, None, s, 0, None), "null")):
        assert call(*args) == rt.GR_E_ARG and msg in rt.last_error(), (msg, rt.last_error())


def test_append_refuses_a_rotation_of_another_head_dim():
    rt, d, cache, batch, spec = _parts()
    spec.head_dim = 128
    p, s = ctypes.addressof, rt._ll3(256, 64, 64)
    rc = rt.lib().gr_paged_append(p(cache), p(batch), p(spec), None, None, 0, None, None, d, d, s, s, None, None, None)
    assert rc == rt.GR_E_ARG and "head dim" in rt.last_error()


def test_workspace_is_what_the_parts_need():
    rt, d, cache, batch, spec = _parts()
    size = rt.lib().gr_paged_attn_workspace
    batch.B, batch.width = 1, 4096                      # one sequence of up to 65,536 keys: shared out
    one = size(ctypes.addressof(cache), ctypes.addressof(batch), 8)
    assert one > 0 and one % (2 * 32 * 66 * 4) == 0     # two tiles of 32 rows x (64 + 2) floats a workgroup
    batch.max_len = 200                                 # too few keys to share
    assert size(ctypes.addressof(cache), ctypes.addressof(batch), 8) == 0


def test_rotary_tables():
    from grammar.rotary import Rotary
    r = Rotary(64, rotary_dim=48, sections=[4, 8, 12], base=500.0, device="cpu")
    assert r.axes.tolist() == [0] * 4 + [1] * 8 + [2] * 12
    for j, (f, t) in enumerate(zip(r.inv_freq, r.turns.tolist())):
        assert f == 500.0 ** -(j / 24)
        assert abs(t % (1 << 64) / 2 ** 64 - f / (2 * math.pi)) <= 2.0 ** -53
    per = Rotary(64, rotary_dim=48, sections=[4, 8, 12], base=500.0, per_axis=True, device="cpu")
    assert per.inv_freq[4] == per.inv_freq[12] == 1.0 and per.inv_freq[3] == 500.0 ** -0.75
    own = Rotary(32, inv_freq=torch.linspace(0, 9, 16), device="cpu")
    assert own.inv_freq[15] == 9.0 and abs(own.turns[15].item() % (1 << 64) / 2 ** 64 - (9 / (2 * math.pi)) % 1) <= 2.0 ** -52


@pytest.mark.parametrize("kw", [dict(head_dim=40), dict(head_dim=512), dict(head_dim=64, rotary_dim=40),
                                dict(head_dim=64, rotary_dim=80), dict(head_dim=64, rotary_dim=0),
                                dict(head_dim=64, sections=[16, 15]), dict(head_dim=64, sections=[-1, 33]),
                                dict(head_dim=64, sections=[]), dict(head_dim=64, sections=[4] * 8 + [0]),
                                dict(head_dim=64, base=0.0), dict(head_dim=64, inv_freq=[1.0] * 31),
                                dict(head_dim=64, inv_freq=[float("inf")] * 32)])
def test_bad_rotary_settings_are_refused(kw):
    from grammar.rotary import Rotary
    with pytest.raises(ValueError):
        Rotary(**kw, device="cpu")


def test_cpu_tensors_are_refused():
    from grammar.paged import PagedCache
    with pytest.raises(ValueError, match="GPU"):
        PagedCache.empty(4, 2, 16, 64, torch.float16, device="cpu")
