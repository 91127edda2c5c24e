"""What calls on normed heads and quantised caches return on a given stream is memory of that stream."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_result_streams_gpu import _cuda, _heads, test_results_belong_to_the_launch_stream as _belongs  # noqa: E402


def _normed():
    from grammar.norm import HeadNorm
    from grammar.rotary import Rotary
    w = 1 + 0.2 * torch.randn(64, device="cuda")
    return Rotary(64), HeadNorm(w, w.flip(0)), torch.arange(256, dtype=torch.int32, device="cuda")


def _norm_rotary(stream):
    from grammar.norm import norm_rotary_fwd
    rot, norm, pos = _normed()
    q, k = _heads(2, 96, 256, 64), _heads(2, 48, 256, 64)
    return lambda: norm_rotary_fwd(q, k, pos, rot, norm, stream=stream)


def _norm_rotary_bwd(stream):
    from grammar.norm import norm_rotary_bwd
    rot, norm, pos = _normed()
    q, k = _heads(2, 96, 256, 64), _heads(2, 48, 256, 64)
    return lambda: norm_rotary_bwd(q, k, pos, rot, norm, q, k, stream=stream)


def _quantised(stream, what):
    from grammar.paged import QuantizedPagedCache, paged_append, paged_attention, paged_read
    rot, norm, _ = _normed()
    cache = QuantizedPagedCache.empty(64, 8, 16, 64, torch.float16)
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(4, 16)
    lens = torch.full((4,), 256, dtype=torch.int32, device="cuda")
    q, k = _heads(4, 64, 256, 64), _heads(4, 8, 256, 64)
    paged_append(k, k, cache, table, lens, norm=norm)
    if what == "append":
        return lambda: paged_append(k, k, cache, table, lens, q=q, rotary=rot, norm=norm, stream=stream)
    if what == "read":
        return lambda: paged_read(cache, table, lens, 300, stream=stream)
    return lambda: paged_attention(q, cache, table, lens, stream=stream)


def _append(stream):
    return _quantised(stream, "append")


def _attention(stream):
    return _quantised(stream, "attend")


def _read(stream):
    return _quantised(stream, "read")


@pytest.mark.parametrize("raw", [False, True], ids=["stream", "handle"])
@pytest.mark.parametrize("call", [_norm_rotary, _norm_rotary_bwd, _append, _attention, _read], ids=lambda f: f.__name__[1:])
def test_results_of_normed_heads_and_quantised_caches(call, raw):
    _cuda()
    _belongs(call, raw)
