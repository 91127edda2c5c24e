"""What a call on a given stream returns is memory of that stream, and safe to be
read and dropped on the current one."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def _rotary(stream):
    from grammar.rotary import Rotary, rotary_fwd
    rot = Rotary(64)
    q, k, pos = torch.randn(2, 96, 256, 64, device="cuda").half(), torch.randn(2, 48, 256, 64, device="cuda").half(), \
        torch.arange(256, dtype=torch.int32, device="cuda")
    return lambda: rotary_fwd(q, k, pos, rot, stream=stream)


def _paged(stream, attend):
    from grammar.paged import PagedCache, paged_append, paged_attention
    from grammar.rotary import Rotary
    rot, cache = Rotary(64), PagedCache(*(torch.randn(64, 8, 16, 64, device="cuda").half() for _ in range(2)))
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(4, 16)
    lens = torch.full((4,), 256, dtype=torch.int32, device="cuda")
    q, k = torch.randn(4, 64, 256, 64, device="cuda").half(), torch.randn(4, 8, 256, 64, device="cuda").half()
    if attend:
        return lambda: paged_attention(q, cache, table, lens, stream=stream)
    return lambda: paged_append(k, k, cache, table, lens, q=q, rotary=rot, stream=stream)


def _paged_append(stream):
    return _paged(stream, False)


def _paged_attention(stream):
    return _paged(stream, True)


def _heads(*shape):
    return torch.randn(*shape, device="cuda").half()


def _flash(stream):
    from grammar.attention import flash_attention_fwd
    q = _heads(2, 8, 1024, 64)
    return lambda: flash_attention_fwd(q, q, q, stream=stream)


def _flash_train(stream):
    from grammar.attention import flash_attention_fwd_train
    q = _heads(2, 8, 1024, 64)
    return lambda: flash_attention_fwd_train(q, q, q, stream=stream)


def _flash_bwd(stream):
    from grammar.attention import flash_attention_bwd, flash_attention_fwd_train
    q = _heads(2, 8, 1024, 64)
    o, lse = flash_attention_fwd_train(q, q, q)
    return lambda: flash_attention_bwd(q, q, q, o, o, lse, stream=stream)


def _decode(stream):
    from grammar.attention import flash_attention_decode
    q, kv = _heads(4, 64, 64, 128), _heads(4, 64, 256, 128)
    return lambda: flash_attention_decode(q, kv, kv, stream=stream)


def _bound_decode(stream):
    from grammar.attention import bind_flash_attention_decode_noalloc
    q, kv = _heads(4, 64, 64, 128), _heads(4, 64, 256, 128)
    return lambda: bind_flash_attention_decode_noalloc(q, kv, kv, splits=1, stream=stream)[0]()


def _gemm(stream):
    from grammar.gemm import gemm
    a, b = _heads(1024, 256), _heads(256, 2048)
    return lambda: gemm(a, b, stream=stream)


def _mlp(stream):
    from grammar.gemm import mlp_fwd
    x, w1, w2 = _heads(2048, 1024), _heads(1024, 512) / 16, _heads(512, 1024) / 16
    return lambda: mlp_fwd(x, w1, w2, stream=stream)


CALLS = [_rotary, _paged_append, _paged_attention, _flash, _flash_train, _flash_bwd, _decode, _bound_decode, _gemm, _mlp]


def _stream_of(t):
    """The handle of the stream whose pool a tensor's memory is from."""
    return next(seg["stream"] for seg in torch.cuda.memory_snapshot()
                if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"])


@pytest.mark.parametrize("raw", [False, True], ids=["stream", "handle"])
@pytest.mark.parametrize("call", CALLS, ids=lambda f: f.__name__[1:])
def test_results_belong_to_the_launch_stream(call, raw):
    """A result is memory of the stream that its launch writes it on: no work of another stream can still be reading
    what was there before. Dropped, it also waits for what the current stream has queued by then."""
    _cuda()
    side = torch.cuda.Stream()
    print(f"[case] results of {call.__name__} raw={raw}", flush=True)
    torch.manual_seed(4)
    want = call(None)()
    torch.manual_seed(4)
    run = call(side.cuda_stream if raw else side)
    torch.cuda.synchronize()
    got = run()
    want, got = (x if isinstance(x, tuple) else (x,) for x in (want, got))
    torch.cuda.current_stream().wait_stream(side)
    for g, w in zip(got, want):
        assert torch.equal(g, w) and g.stride() == w.stride()
        assert _stream_of(g) == side.cuda_stream and _stream_of(w) == 0
    at, size = [g.data_ptr() for g in got], [g.numel() * g.element_size() for g in got]
    torch.cuda._sleep(50_000_000)
    copies = [g.clone() for g in got]                        # queued behind the wait
    del g, got
    with torch.cuda.stream(side):
        new = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in size]
    assert not torch.cuda.current_stream().query()
    assert not set(at) & {t.data_ptr() for t in new}
    assert all(torch.equal(c, w) for c, w in zip(copies, want))
