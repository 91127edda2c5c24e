"""What the numbers of a quantised cache stand for: numbers below the tokens' type's normal range, the bounds of what
quantising loses, keys that a norm made small, and norm weights in fp32."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_norm_gpu import FWD, _normed  # noqa: E402
from test_paged_gpu import APPENDS, _cuda, _rotated  # noqa: E402
from test_paged8_gpu import E4M3, E8M0, _check_rows, _dequantised, _scale_of, test_append as _append  # noqa: E402

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
# scale exponents about the least under which the type holds every number, and that least: fp16's and bf16's smallest
# steps are 2^-24 and 2^-133, e4m3's 2^-9
SCALES = {"fp16": (range(-26, -10), -15), "bf16": (range(-127, -111), -124)}


def _small(dtype, heads, dev):
    """A cache of 64 pages whose first slots' values are all 256 bytes, 4 pages of 64 dims to a scale, and the numbers
    they stand for, [16 scales, 256]."""
    from grammar.paged import QuantizedPagedCache
    ks, _ = SCALES[dtype]
    v = torch.arange(256, dtype=torch.uint8, device=dev).view(1, 4, 1, 1, 64).expand(16, 4, heads, 16, 64).reshape(64, heads, 16, 64)
    sb = torch.full((64, heads, 2, 16), 127, dtype=torch.uint8, device=dev)
    sb[:, :, 1] = torch.tensor([127 + k for k in ks], dtype=torch.uint8, device=dev).repeat_interleave(4).view(64, 1, 1)
    cache = QuantizedPagedCache(torch.zeros_like(v).view(E4M3), v.contiguous().view(E4M3), sb.view(E8M0), DT[dtype])
    stand = _dequantised(cache.v[:, 0, 0], sb[:, 0, 1, 0].contiguous().view(E8M0)).view(16, 256)
    table = torch.arange(64, dtype=torch.int32, device=dev).view(64, 1)
    return cache, stand, table, torch.ones(64, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_numbers_below_the_normal_range_round_once_more(dtype):
    """Read back and attended, a number times its scale is the nearest of the tokens' type (to even): itself, but for
    scales below the least under which the type holds them all, where it is a whole number of the type's smallest steps."""
    from grammar.paged import paged_attention, paged_read
    dev, dt, (ks, least) = _cuda(), DT[dtype], SCALES[dtype]
    step = 2.0 ** -24 if dtype == "fp16" else 2.0 ** -133
    cache, stand, table, lens = _small(dtype, 5, dev)
    held = ~stand.isnan()
    # the definition: nearest whole number of steps, ties to even (torch.round), below 2^10 or 2^7 steps; else exact
    want = torch.where(stand.abs() < step * (1024 if dtype == "fp16" else 128), torch.round(stand / step) * step, stand)
    rounded = ((want != stand) & held).sum(1).tolist()
    assert [n > 0 for n in rounded] == [k < least for k in ks]
    if dtype == "fp16":
        assert rounded[list(ks).index(-17)] == 2 * 16                # of 2 x 127 numbers
    # one key: its weight is 1 and the result its value, in tiles of 16, 32 and 128 rows
    results = [paged_read(cache, table, lens, 1)[1].view(16, 4, 5, 64)]
    for n in (1, 40, 100):
        o = paged_attention(torch.zeros((64, 5, n, 64), device=dev, dtype=dt), cache, table, lens, causal=False)
        results += [o[:, :, i].view(16, 4, 5, 64) for i in (0, n - 1)]
    for got in results:
        for h in range(5):
            x = got[:, :, h].reshape(16, 256)
            assert torch.equal(x.isnan(), stand.isnan()) and torch.equal(x[held].double(), want[held])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_what_quantising_loses(dtype, D):
    """2^-4 of an element at most, or 2^-10 of the scale, which is 2^-17.8 of the row's largest magnitude; the latter in
    full by a row of 225 and nearly 1.5 steps."""
    from grammar.paged import QuantizedPagedCache, paged_append, paged_read
    dev, dt = _cuda(), DT[dtype]
    g = torch.Generator("cpu").manual_seed(D)
    x = torch.randn((1, 4, 300, D), generator=g) * torch.exp2(4 * torch.randn((1, 4, 300, D), generator=g))
    x *= torch.exp2(torch.randint(-4, 5, (1, 4, 300, 1), generator=g).float())
    x = x.clamp(-60000, 60000)
    x[0, 0, 0] = 0
    x[0, 0, 0, 0], x[0, 0, 0, 1] = 225, 3 * 2.0 ** -10 * (1 - 2.0 ** -8)
    x = x.to(dt).to(dev)
    cache = QuantizedPagedCache.empty(20, 4, 16, D, dt)
    table, lens = torch.arange(20, dtype=torch.int32, device=dev).view(1, 20), torch.tensor([300], dtype=torch.int32, device=dev)
    paged_append(x, x, cache, table, lens)
    top = x.double().abs().amax(-1, keepdim=True)
    scale = torch.exp2(_scale_of(top).double() - 127)
    for got in paged_read(cache, table, lens, 300):
        off = (got.double() - x.double()).abs()
        assert (off <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * scale)).all()
        assert (off <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -17.8 * top)).all()
        assert off[0, 0, 0, 1] > 2.0 ** -18 * top[0, 0, 0, 0]         # not within half of 2^-17 of the largest


@pytest.mark.parametrize("dtype,power", [("fp16", -9), ("fp16", -14), ("bf16", -9)])
@pytest.mark.parametrize("rotated", [True, False])
def test_keys_that_a_norm_makes_small(dtype, power, rotated):
    """Weights of about 2^power: the stored rows are the definition's, whatever the tokens' type holds, and are read back
    as the nearest numbers that it does."""
    from grammar.norm import HeadNorm
    from grammar.paged import QuantizedPagedCache, paged_append, paged_read
    from grammar.rotary import Rotary
    dev, dt = _cuda(), DT[dtype]
    D, N, H = 128, 200, 3
    g = torch.Generator("cpu").manual_seed(3)
    k = torch.randn((1, H, N, D), generator=g).to(dt).to(dev)
    w = ((1 + 0.3 * torch.randn(D, generator=g)) * 2.0 ** power).to(dev)
    norm = HeadNorm(w, w, eps=1e-6)
    rot = Rotary(D, device=dev) if rotated else None
    cache = QuantizedPagedCache.empty(13, H, 16, D, dt)
    table, lens = torch.arange(13, dtype=torch.int32, device=dev).view(1, 13), torch.tensor([N], dtype=torch.int32, device=dev)
    paged_append(k, k, cache, table, lens, norm=norm, rotary=rot)
    y, size = _normed(k, w, norm.eps)[0][0], None
    if rotated:
        y, size = _rotated(y.transpose(0, 1), torch.arange(N, device=dev), rot)
        y, size = y.transpose(0, 1), size.transpose(0, 1)
    size = y.abs() if size is None else size
    q, sb = (t.view(torch.uint8).transpose(0, 1).flatten(1, 2)[:, :N] for t in (cache.k, cache.scales[:, :, 0]))
    _check_rows(q.contiguous().view(E4M3), sb, y, size, FWD, dt, "keys")
    stand = _dequantised(q.contiguous().view(E4M3), sb.contiguous().view(E8M0))
    assert (dtype == "fp16") == bool((stand.to(dt).double() != stand).any())
    assert torch.equal(paged_read(cache, table, lens, N)[0][0], stand.float().to(dt))


@pytest.mark.parametrize("news,lens,Hq,Hkv,D,S,rd,sections,inter,dtype,ragged", APPENDS)
def test_append_with_fp32_weights(news, lens, Hq, Hkv, D, S, rd, sections, inter, dtype, ragged):
    _append(news, lens, Hq, Hkv, D, S, rd, sections, inter, dtype, ragged, "fp32", True)
