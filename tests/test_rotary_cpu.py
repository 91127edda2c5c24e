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
