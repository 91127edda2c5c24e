"""The Python side of the position rotation that needs no GPU."""
import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    """rotary() with a stand-in for the launch: copies, like a kernel's, that autograd knows nothing of."""
    from grammar import rotary as R
    made = []

    def stand_in(q, k, positions, rot, *, inverse=False):
        made.append(inverse)
        return q.detach().clone(), None if k is None else k.detach().clone()
    monkeypatch.setattr(R, "rotary_fwd", stand_in)
    return made


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(launches, which, grad):
    """A tangent would be lost in the launch: it raises, recorded or not, as flash_attention does."""
    import torch.autograd.forward_ad as forward_ad
    from grammar.rotary import rotary
    q, k = torch.randn(1, 2, 4, 64), torch.randn(1, 1, 4, 64)
    pos = torch.arange(4, dtype=torch.int32)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = {"q": q, "k": k}
        dual[which] = forward_ad.make_dual(dual[which], torch.ones_like(dual[which]))
        with pytest.raises(NotImplementedError):
            rotary(dual["q"], dual["k"], pos, None)
        plain = rotary(q, k, pos, None)                     # no tangent in the level: one launch
        assert torch.equal(plain[0], q) and torch.equal(plain[1], k)
    assert rotary(q, None, pos, None)[1] is None
    assert launches[-2:] == [False, False]


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle", "save"])
def test_rotary_can_be_copied_and_pickled(how):
    """As part of a model that is copied or saved whole; a copy points at tables of its own."""
    import copy
    import io
    import pickle
    from grammar.rotary import Rotary
    r = Rotary(64, rotary_dim=48, sections=[4, 8, 12], base=500.0, interleaved=True, device="cpu")

    def saved(x):
        file = io.BytesIO()
        torch.save({"rotary": x}, file)
        file.seek(0)
        return torch.load(file, weights_only=False)["rotary"]          # (its own file, just written)
    c = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x)),
         "save": saved}[how](r)
    assert type(c) is Rotary and c is not r and c.ref != r.ref
    for name in ("head_dim", "rotary_dim", "interleaved", "sections", "naxes", "inv_freq", "device", "index"):
        assert getattr(c, name) == getattr(r, name), name
    assert torch.equal(c.turns, r.turns) and torch.equal(c.axes, r.axes)
    assert c.desc.turns == c.turns.data_ptr() and c.desc.axes == c.axes.data_ptr()
    assert how == "copy" or c.turns.data_ptr() != r.turns.data_ptr()
    assert (c.desc.pairs, c.desc.naxes, c.desc.head_dim, c.desc.interleaved) == (24, 3, 64, 1)


def test_turns_are_the_nearest_to_the_frequency():
    """To a unit of 2^-64 turns, against 60-digit decimals (pi by its published digits), for tiny and huge ones too."""
    import math
    from decimal import Decimal, getcontext
    from grammar.rotary import Rotary
    getcontext().prec = 120
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")
    freqs = [1.0, 0.5, 10000.0 ** -0.25, 500.0 ** -0.9, math.pi, 2 * math.pi, 1e-30, 5e-324, -1.0, -1e-9, 9.0, 12345.678,
             2.0 ** 53, 1e15, -1e15, 0.0]
    r = Rotary(32, inv_freq=freqs, device="cpu")
    for f, t in zip(freqs, r.turns.tolist()):
        want = Decimal(f) / (2 * pi) * 2 ** 64
        off = (Decimal(t) - want) % 2 ** 64
        assert min(abs(off), abs(2 ** 64 - abs(off))) <= Decimal("0.51"), (f, t, off)
    assert Rotary(32, inv_freq=[1e308] * 16, device="cpu").inv_freq[0] == 1e308


def test_sizes_past_32_bits_are_refused():
    """The library takes 32-bit counts, and ctypes would pass 2^32 + 5 tokens as 5. (A head of 16 in fp16 is 32 bytes:
    such tensors fit a GPU. Shapes alone here.)"""
    from grammar.paged import _batch_sizes
    from grammar.rotary import Rotary, _tokens, rotary_fwd
    n = 2 ** 32 + 5
    for shape, st in (((1, 1, n, 16), (n * 16, 16, 16, 1)), ((n, 1, 1, 16), (16, 16, 16, 1)), ((1, n, 1, 16), (0, 16, 0, 1)),
                      ((2 ** 16, 1, 2 ** 16, 16), (2 ** 20, 16, 16, 1)), ((1, 1, 2 ** 31, 16), (0, 0, 16, 1))):
        assert _tokens(shape, st, None, None, 16) == "too many"
        assert _tokens((shape[0], 1, shape[2], 16), st, shape, st, 16) == "too many"
    assert _tokens((1, 1, 2 ** 31 - 1, 16), (0, 0, 16, 1), None, None, 16)[:3] == (1, 2 ** 31 - 1, 1)
    for table, x in (((1, n), (1, 1, 1, 64)), ((1, 4), (1, 1, n, 64)), ((1, 4), (1, n, 1, 64)), ((n, 4), (n, 1, 1, 64))):
        assert "too large" in _batch_sizes(table, (table[1], 1), (table[0],), (1,), None, None, x)
    assert "too large" in _batch_sizes((1, 4), (4, 1), (1,), (1,), (2,), (1,), (n, 1, 64))

    class Far:                                                        # the shape of a tensor that no test can hold
        shape, dtype = torch.Size((1, 1, n, 16)), torch.float16
        stride = staticmethod(lambda: (0, 0, 16, 1))
        get_device = staticmethod(lambda: 0)
    rot = Rotary(16, device="cpu")
    rot.index = 0
    with pytest.raises(ValueError, match="too many tokens"):
        rotary_fwd(Far(), None, None, rot)
