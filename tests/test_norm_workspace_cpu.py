"""The workspace of the gradient of normed heads is sized by the heads' own GPU (no GPU: the library's answer is a stand-in's)."""
import contextlib


def test_the_size_is_asked_for_on_the_heads_gpu(monkeypatch):
    import torch
    from grammar import norm as gn
    now, cus = [0], {0: 256, 1: 64, 2: 304}

    @contextlib.contextmanager
    def device(index):
        before, now[0] = now[0], index
        yield
        now[0] = before

    class Library:
        @staticmethod
        def gr_norm_rotary_bwd_workspace(*sizes):
            assert sizes == (32, 8, 128, 2, 4096)
            return cus[now[0]] * 4096
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(gn.rt, "lib", lambda: Library)
    gn._bwd_workspace.cache_clear()
    try:
        for index in (1, 0, 2, 1):                                    # the current one is 0 all the time
            assert gn._bwd_workspace(index, 32, 8, 128, 2, 4096) == cus[index] * 4096
        assert now == [0]
    finally:
        gn._bwd_workspace.cache_clear()
