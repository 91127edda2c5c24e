"""The operators of cached and positioned attention that this framework's speed
is judged by: the position rotation of queries and keys (one or several axes)
with its gradient, appending new keys and values to a paged cache with the
rotation on the way, and attention of new tokens over that cache.

listed() gives the fixed cases, draw() more of the same ranges. prepare()
makes what a program holds before the call, run() is one pass, with plain torch
operations where `own` is false and through the framework's entry points where
it is true, and exact() is the same result in 64 bits from the definition.

Shapes. A case has `B` sequences with `Hq` query and `Hkv` key/value heads of
`D`. Uniform batches are [B, heads, tokens, D]; ragged ones are packed, [tokens
of all sequences, heads, D], with the first row of each sequence in `starts`,
and may have rows behind the last sequence (a batch padded to a fixed size),
which no operator writes. The cache is pages of `S` tokens, [pages, Hkv, S, D];
`table` names each sequence's pages in order, `lens` counts its keys, the new
tokens' among them, so that new token i of n stands at position len - n + i."""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ELEM = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed() -> list:
    return [
        # queries and keys of one short sequence, forward only: the smallest rotation, where latency counts
        {"name": "rotary_short", "kind": "rotary", "B": 1, "N": 320, "Hq": 4, "Hkv": 4, "D": 64, "rd": 64,
         "axes": 1, "per_axis": False, "interleaved": False, "train": False, "far": 0, "dtype": "bf16"},
        # a training step's rotation in an encoder of images or video: time, height and width, an odd token count,
        # each axis with frequencies of its own
        {"name": "rotary_video_train", "kind": "rotary", "B": 3, "N": 1571, "Hq": 16, "Hkv": 16, "D": 64, "rd": 64,
         "axes": 3, "per_axis": True, "interleaved": True, "train": True, "far": 0, "dtype": "fp16"},
        # a training step's rotation at the size of the benchmark's long attention: 4,096 tokens, 32 heads of 128
        {"name": "rotary_long_train", "kind": "rotary", "B": 2, "N": 4096, "Hq": 32, "Hkv": 32, "D": 128, "rd": 128,
         "axes": 1, "per_axis": False, "interleaved": False, "train": True, "far": 0, "dtype": "bf16"},
        # one decode step of a batch: every sequence's new key and value into its page, its query rotated
        {"name": "append_step", "kind": "append", "B": 24, "new": 1, "long": 24, "pad": 0, "lo": 90, "hi": 900,
         "Hq": 32, "Hkv": 8, "D": 128, "S": 16, "rd": 128, "axes": 1, "interleaved": False, "ragged": False,
         "mix": 1, "dtype": "bf16"},
        # a server's mixed step: two prompts' chunks among decoding sequences, half of each head rotated, padded batch
        {"name": "append_mixed", "kind": "append", "B": 19, "new": 423, "long": 2, "pad": 17, "lo": 500, "hi": 2500,
         "Hq": 16, "Hkv": 16, "D": 64, "S": 32, "rd": 32, "axes": 1, "interleaved": True, "ragged": True,
         "mix": 2, "dtype": "fp16"},
        # whole prompts with images, positions on three axes
        {"name": "append_prompts", "kind": "append", "B": 3, "new": 2731, "long": 3, "pad": 0, "lo": 2731, "hi": 4000,
         "Hq": 32, "Hkv": 8, "D": 128, "S": 64, "rd": 128, "axes": 3, "interleaved": False, "ragged": True,
         "mix": 3, "dtype": "bf16"},
        # one token of one short conversation: the smallest attention, where latency counts
        {"name": "decode_one", "kind": "attend", "B": 1, "new": 1, "long": 1, "pad": 0, "lo": 419, "hi": 419,
         "Hq": 16, "Hkv": 16, "D": 64, "S": 16, "causal": True, "ragged": False, "mix": 4, "dtype": "fp16"},
        # a decode step of a full batch with contexts of all lengths
        {"name": "decode_batch", "kind": "attend", "B": 48, "new": 1, "long": 48, "pad": 0, "lo": 150, "hi": 8000,
         "Hq": 32, "Hkv": 8, "D": 128, "S": 16, "causal": True, "ragged": False, "mix": 5, "dtype": "bf16"},
        # two long contexts, 16 query heads to a key head
        {"name": "decode_long", "kind": "attend", "B": 2, "new": 1, "long": 2, "pad": 0, "lo": 70001, "hi": 131009,
         "Hq": 32, "Hkv": 2, "D": 128, "S": 128, "causal": True, "ragged": False, "mix": 6, "dtype": "fp16"},
        # five drafted tokens a sequence to verify, seven query heads to a key head
        {"name": "drafted_tokens", "kind": "attend", "B": 16, "new": 5, "long": 16, "pad": 0, "lo": 300, "hi": 4100,
         "Hq": 28, "Hkv": 4, "D": 128, "S": 32, "causal": True, "ragged": False, "mix": 7, "dtype": "bf16"},
        # the server's mixed step: two prompts' chunks among decoding sequences, padded batch
        {"name": "chunk_mixed", "kind": "attend", "B": 19, "new": 423, "long": 2, "pad": 17, "lo": 500, "hi": 2500,
         "Hq": 16, "Hkv": 16, "D": 64, "S": 32, "causal": True, "ragged": True, "mix": 2, "dtype": "fp16"},
        # a long prompt's second chunk of 4,096 tokens onto the 4,096 that are cached
        {"name": "chunk_long", "kind": "attend", "B": 1, "new": 4096, "long": 1, "pad": 0, "lo": 8192, "hi": 8192,
         "Hq": 32, "Hkv": 8, "D": 128, "S": 64, "causal": True, "ragged": True, "mix": 8, "dtype": "bf16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(("rotary", "append", "attend", "attend"))
    d = rng.choice((64, 128))
    half = rng.choice(("fp16", "bf16"))
    hkv = _log(rng, 1, 16)
    hq = hkv * rng.choice((1, 1, 2, 4, 5, 8))
    axes = rng.choice((1, 1, 2, 3))
    rd = rng.choice((d, d, d // 2))
    if kind == "rotary":
        c = {"kind": kind, "B": _log(rng, 1, 4), "N": _log(rng, 1, 4096), "Hq": min(hq, 32), "Hkv": hkv, "D": d,
             "rd": rd, "axes": axes, "per_axis": axes > 1 and rng.random() < 0.5, "interleaved": rng.random() < 0.4,
             "train": rng.random() < 0.6, "far": rng.choice((0, 0, 200_000)), "dtype": rng.choice((half, half, "fp32"))}
        while work(c)["bytes"] > 1.0e9:
            c["N"] = max(1, c["N"] // 2)
        return c
    s = rng.choice((16, 32, 64, 128))
    b = _log(rng, 1, 64)
    u = rng.random()
    if u < 0.45:                                   # a decode step
        new, n_long, ragged, pad = 1, b, rng.random() < 0.3, 0
    elif u < 0.6:                                  # a few tokens each
        new, n_long, ragged, pad = _log(rng, 2, 16), b, False, 0
    elif u < 0.85:                                 # a mixed step
        new, n_long, ragged, pad = _log(rng, 17, 2048), min(b, rng.choice((1, 2))), True, rng.choice((0, 5, 31))
    else:                                          # whole chunks
        b = min(b, 3)
        new, n_long, ragged, pad = _log(rng, 17, 4096), b, True, 0
    lo = max(new, _log(rng, 1, 4096))
    hi = max(lo, min(16384, lo * rng.choice((1, 2, 4, 8))))
    c = {"kind": kind, "B": b, "new": new, "long": n_long, "pad": pad, "lo": lo, "hi": hi, "Hq": hq, "Hkv": hkv,
         "D": d, "S": s, "ragged": ragged, "mix": rng.randrange(1, 10_000), "dtype": half}
    if kind == "append":
        c.update(rd=rd, axes=axes, interleaved=rng.random() < 0.4)
        c["hi"] = max(c["lo"], min(c["hi"], 4096))
        while _cache_bytes(c) > 1.0e9 or work(c)["bytes"] > 2.0e8:
            c["B"], c["long"] = max(1, c["B"] // 2), max(1, c["long"] // 2)
            c["new"], c["lo"], c["hi"] = max(1, c["new"] // 2), max(1, c["lo"] // 2), max(1, c["hi"] // 2)
        return c
    c["causal"] = rng.random() < 0.8
    while _cache_bytes(c) > 1.0e9 or work(c)["flops"] > 4.0e11:
        c["B"], c["long"] = max(1, c["B"] // 2), max(1, c["long"] // 2)
        if c["B"] == 1:
            c["new"], c["lo"], c["hi"] = max(1, c["new"] // 2), max(1, c["lo"] // 2), max(1, c["hi"] // 2)
    return c


def _sequences(case: dict) -> tuple:
    """(new tokens, keys) of each sequence: `long` of them bring `new` tokens, the others one; the key counts are
    spread over [lo, hi]."""
    rng = random.Random(case["mix"])
    news = [case["new"] if b < case["long"] else 1 for b in range(case["B"])]
    if case["ragged"]:
        rng.shuffle(news)
    return news, [max(n, rng.randint(case["lo"], case["hi"])) for n in news]


def _cache_bytes(case: dict) -> int:
    return 2 * sum(_sequences(case)[1]) * case["Hkv"] * case["D"] * ELEM[case["dtype"]]


def work(case: dict) -> dict:
    e, d, hq, hkv = ELEM[case["dtype"]], case["D"], case["Hq"], case["Hkv"]
    if case["kind"] == "rotary":
        # q and k in, rotated out, and as much again for the gradients; a pair is four products and two sums
        tokens, passes = case["B"] * case["N"], 2 if case["train"] else 1
        return {"bytes": passes * (2 * e * tokens * (hq + hkv) * d + 4 * case["axes"] * case["N"]),
                "flops": passes * 3 * tokens * (hq + hkv) * case["rd"]}
    news, lens = _sequences(case)
    t = sum(news)
    if case["kind"] == "append":
        # q in and out, k and v in and into their pages
        return {"bytes": 2 * e * t * (hq + 2 * hkv) * d, "flops": 3 * t * (hq + hkv) * case["rd"]}
    # every live key and value once, q in and the result out; two products over the visible pairs
    pairs = sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for n, m in zip(news, lens))
    return {"bytes": e * (2 * sum(lens) * hkv * d + 2 * t * hq * d), "flops": 4 * hq * d * pairs}


def _sections(case: dict) -> list:
    """Rotated pairs of each axis: even shares, the last axis taking the rest."""
    pairs, axes = case["rd"] // 2, case["axes"]
    share = pairs // axes
    return [share] * (axes - 1) + [pairs - share * (axes - 1)]


def _inputs(case: dict, seed: int) -> dict:
    """The case's tensors, from the seed alone: activations and cached entries N(0, 1) in the storage type. Pages
    are handed out in no order, as a cache in use has them."""
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    def ints(hi, *shape):
        return torch.randint(0, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "rotary":
        N, A = case["N"], case["axes"]
        far = case["far"] + int(ints(64, 1))
        n = torch.arange(N, device="cuda", dtype=torch.int32)
        if A == 1:
            pos = n + far
        else:                                       # a grid of patches in reading order, axis by axis
            side = max(1, round(N ** (1 / A)))
            pos = torch.stack([n // side ** (A - 1 - a) % (side if a else N + 1) + far for a in range(A)]).contiguous()
        s = {"pos": pos}
        for name, h in (("q", Hq), ("k", Hkv), ("dq", Hq), ("dk", Hkv)):
            # activations [B, N, heads, D], as a projection leaves them
            s[name] = randn(B, N, h, D)
        return s
    news, lens = _sequences(case)
    S = case["S"]
    pages = [-(-m // S) for m in lens]
    total, width = sum(pages) + 3, max(pages)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    s = {"k_pages": randn(total, Hkv, S, D), "v_pages": randn(total, Hkv, S, D), "table": table,
         "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "news_host": news, "lens_host": lens}
    T = sum(news) + case["pad"]
    if case["kind"] == "attend":
        s["q"] = randn(T, Hq, D) if case["ragged"] else randn(B, Hq, case["new"], D)
    else:
        # one projection's rows hold q, k and v next to each other: strided views
        rows = randn(T, Hq + 2 * Hkv, D)
        if not case["ragged"]:
            rows = rows.view(B, case["new"], Hq + 2 * Hkv, D).transpose(1, 2)
        h = 1
        s["q"], s["k"], s["v"] = rows.split([Hq, Hkv, Hkv], dim=h)
        if case["axes"] > 1:                        # text runs along all axes, an image along two
            base = torch.cat([torch.arange(m - n, m, dtype=torch.int32) for n, m in zip(news, lens)]
                             + [torch.zeros(case["pad"], dtype=torch.int32)]).cuda()
            pos = torch.stack([base] + [base + ints(40, T) for _ in range(case["axes"] - 1)]).contiguous()
            s["pos"] = pos if case["ragged"] else pos.view(case["axes"], B, case["new"])
    if case["ragged"]:
        ends = [0]
        for n in news:
            ends.append(ends[-1] + n)
        s["starts"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    return s


def _inv_freq(case: dict) -> tuple:
    """(frequency in radians a position, axis) of each rotated pair, float64."""
    base, freq, axis = 10000.0, [], []
    for a, count in enumerate(_sections(case)):
        for j in range(count):
            x = j / count if case.get("per_axis") else len(freq) / (case["rd"] // 2)
            freq.append(base ** -x)
            axis.append(a)
    return torch.tensor(freq, dtype=torch.float64, device="cuda"), torch.tensor(axis, device="cuda")


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    s["case"] = case
    kind = case["kind"]
    if kind == "rotary":
        for n in ("q", "k"):
            s[n].requires_grad_(case["train"])
    else:
        s["out"] = torch.zeros_like(s["q"], memory_format=torch.contiguous_format)
    if not own:
        if kind != "attend":
            s["freq"], s["axis"] = _inv_freq(case)
        return s
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cs348k-fast-attention-grammar_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from grammar.paged import PagedCache, bind_paged_append, bind_paged_attention
    from grammar.rotary import Rotary
    if kind != "attend":
        s["rotary"] = Rotary(case["D"], rotary_dim=case["rd"], sections=_sections(case), base=10000.0,
                             per_axis=case.get("per_axis", False), interleaved=case["interleaved"], device="cuda")
    if kind == "rotary":
        return s
    s["cache"] = PagedCache(s["k_pages"], s["v_pages"])
    if case["new"] == 1 and not case["ragged"]:
        # a decode loop runs on fixed buffers: bound once, launched every step
        if kind == "append":
            s["launch"], _ = bind_paged_append(s["k"], s["v"], s["cache"], s["table"], s["lens"], q=s["q"],
                                               rotary=s["rotary"], positions=s.get("pos"), out=s["out"])
        else:
            s["launch"], _ = bind_paged_attention(s["q"], s["cache"], s["table"], s["lens"], causal=case["causal"],
                                                  max_len=max(s["lens_host"]), out=s["out"])
    return s


def run(s: dict):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s: dict):
    from grammar.paged import paged_append, paged_attention
    from grammar.rotary import rotary
    case = s["case"]
    if case["kind"] == "rotary":
        q, k = rotary(s["q"].transpose(1, 2), s["k"].transpose(1, 2), s["pos"], s["rotary"])
        return _rotary_result(s, q, k)
    if "launch" in s:
        s["launch"]()
    elif case["kind"] == "append":
        paged_append(s["k"], s["v"], s["cache"], s["table"], s["lens"], starts=s.get("starts"), q=s["q"],
                     rotary=s["rotary"], positions=s.get("pos"), max_new=case["new"], out=s["out"])
    else:
        paged_attention(s["q"], s["cache"], s["table"], s["lens"], starts=s.get("starts"), causal=case["causal"],
                        max_len=max(s["lens_host"]), max_new=case["new"], out=s["out"])
    return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]} if case["kind"] == "append" else s["out"]


def _rotary_result(s: dict, q, k) -> dict:
    out = {"q": q.detach(), "k": k.detach()}
    if s["case"]["train"]:
        out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]),
                                                   (s["dq"].transpose(1, 2), s["dk"].transpose(1, 2)))
    return out


def _rotate(x, ang, case: dict):
    """x [..., tokens, D] rotated by the angles [..., tokens, pairs], in 32 bits."""
    rd, y = case["rd"], x.float()
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    rot = y[..., :rd]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if case["interleaved"] else (rot[..., :rd // 2], rot[..., rd // 2:])
    u, w = a * cos - b * sin, a * sin + b * cos
    rot = torch.stack((u, w), -1).flatten(-2) if case["interleaved"] else torch.cat((u, w), -1)
    return torch.cat((rot, y[..., rd:]), -1).to(x.dtype)


def _angles(pos, s: dict):
    """Angles [..., pairs] of positions [...] or [axes, ...], in 64 bits: far positions have large angles."""
    p = pos.double().unsqueeze(-1)
    if s["case"]["axes"] == 1:
        return p * s["freq"]
    return torch.cat([p[a] * s["freq"][s["axis"] == a] for a in range(s["case"]["axes"])], -1)


def _run_plain(s: dict):
    case = s["case"]
    if case["kind"] == "rotary":
        ang = _angles(s["pos"], s)
        return _rotary_result(s, _rotate(s["q"].transpose(1, 2), ang, case), _rotate(s["k"].transpose(1, 2), ang, case))
    return _append_plain(s) if case["kind"] == "append" else _attend_plain(s)


def _append_plain(s: dict) -> dict:
    case = s["case"]
    news, S = s["news_host"], case["S"]
    if case["ragged"]:
        t = int(sum(news))
        row = torch.arange(t, device="cuda")
        seq = torch.searchsorted(s["starts"], row, right=True) - 1
        at = s["lens"][seq] - s["starts"][seq + 1] + row           # len - n + i
        q, k, v = s["q"][:t], s["k"][:t], s["v"][:t]
        pos = s["pos"][:, :t] if "pos" in s else at
    else:
        n = case["new"]
        seq = torch.arange(case["B"], device="cuda").repeat_interleave(n)
        at = (s["lens"].unsqueeze(1) - n + torch.arange(n, device="cuda")).flatten()
        q, k, v = (s[x].transpose(1, 2).flatten(0, 1) for x in ("q", "k", "v"))
        pos = s["pos"].flatten(1) if "pos" in s else at
    ang = _angles(pos, s).unsqueeze(1)                               # [tokens, 1, pairs], the heads' alike
    page, slot = s["table"][seq, at // S].long(), at % S
    s["k_pages"][page, :, slot] = _rotate(k, ang, case)
    s["v_pages"][page, :, slot] = v
    q = _rotate(q, ang, case)
    if case["ragged"]:
        s["out"][:q.shape[0]] = q
    else:
        s["out"].copy_(q.view(case["B"], case["new"], case["Hq"], case["D"]).transpose(1, 2))
    return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend_plain(s: dict):
    case = s["case"]
    Hq, Hkv, D, S = case["Hq"], case["Hkv"], case["D"], case["S"]
    group, scale, row = Hq // Hkv, 1.0 / math.sqrt(D), 0
    for b, (n, m) in enumerate(zip(s["news_host"], s["lens_host"])):
        pages = s["table"][b, :-(-m // S)].long()
        k, v = (s[x][pages].transpose(0, 1).flatten(1, 2)[:, :m].float().contiguous() for x in ("k_pages", "v_pages"))
        q = s["q"][row:row + n].transpose(0, 1) if case["ragged"] else s["q"][b]
        o = torch.empty((Hq, n, D), device="cuda")
        kt = k.transpose(1, 2).contiguous()
        step = max(1, int(2 ** 28 // (n * m * group)))               # key heads at a time: bounds the scores' memory
        for h in range(0, Hkv, step):
            c = min(step, Hkv - h)
            qs = q[h * group:(h + c) * group].float().reshape(c, group * n, D)
            sc = torch.matmul(qs, kt[h:h + c]) * scale
            if case["causal"] and n > 1:
                i = torch.arange(n, device="cuda").unsqueeze(1) + (m - n)
                hidden = torch.arange(m, device="cuda").unsqueeze(0) > i
                sc = sc.view(c, group, n, m).masked_fill_(hidden, float("-inf")).view(c, group * n, m)
            p = torch.exp(sc - sc.amax(-1, keepdim=True))
            o[h * group:(h + c) * group] = (torch.matmul(p, v[h:h + c]) / p.sum(-1, keepdim=True)).view(c * group, n, D)
        if case["ragged"]:
            s["out"][row:row + n] = o.transpose(0, 1)
        else:
            s["out"][b] = o
        row += n
    return s["out"]


def _turned(x, pos, case: dict, sign: int = 1):
    """x [tokens, heads, D] in 64 bits, each pair as a complex number times e^(i angle); pos [tokens] or
    [axes, tokens]."""
    x, rd = x.double().clone(), case["rd"]
    pairs = rd // 2
    done = 0
    for a, count in enumerate(_sections(case)):
        p = pos[a] if case["axes"] > 1 else pos
        j = torch.arange(count, dtype=torch.float64, device="cuda")
        x_of = j / count if case.get("per_axis") else (j + done) / pairs
        ang = sign * torch.outer(p.double(), torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), -x_of))
        j = torch.arange(done, done + count, device="cuda")
        first, second = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + pairs)
        z = torch.complex(x[:, :, first], x[:, :, second]) * torch.polar(torch.ones_like(ang), ang).unsqueeze(1)
        x[:, :, first], x[:, :, second] = z.real, z.imag
        done += count
    return x


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    kind, D = case["kind"], case["D"]
    if kind == "rotary":
        def turned(name, sign=1):                   # token rows one sequence after another
            t = s[name]
            pos = s["pos"].repeat(case["B"]) if case["axes"] == 1 else s["pos"].repeat(1, case["B"])
            return _turned(t.flatten(0, 1), pos, case, sign).view(t.shape)
        out = {"q": turned("q").transpose(1, 2), "k": turned("k").transpose(1, 2)}
        if case["train"]:                            # the gradient of a rotation is the rotation back
            out["dq"], out["dk"] = turned("dq", -1), turned("dk", -1)
        return out
    S, row = case["S"], 0
    news, lens = s["news_host"], s["lens_host"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    if kind == "append":
        kc, vc = s["k_pages"].double(), s["v_pages"].double()
    for b, (n, m) in enumerate(zip(news, lens)):
        # the cache slot of every key, in order
        key = torch.arange(m, device="cuda")
        page, slot = s["table"][b].long()[key // S], key % S
        rows = slice(row, row + n)

        def tokens(x):
            return x[rows] if case["ragged"] else x[b].transpose(0, 1)

        def put(o):                                  # o [n, heads, D]
            if case["ragged"]:
                out[rows] = o
            else:
                out[b] = o.transpose(0, 1)
        row += n
        if kind == "append":
            if "pos" in s:
                pos = s["pos"][:, rows] if case["ragged"] else s["pos"][:, b]
            else:
                pos = key[m - n:]
            put(_turned(tokens(s["q"]), pos, case))
            kc[page[m - n:], :, slot[m - n:]] = _turned(tokens(s["k"]), pos, case)
            vc[page[m - n:], :, slot[m - n:]] = tokens(s["v"]).double()
            continue
        q, o = tokens(s["q"]).double(), torch.empty((n, case["Hq"], D), dtype=torch.float64, device="cuda")
        for h in range(case["Hq"]):
            hk = h // (case["Hq"] // case["Hkv"])
            w = q[:, h] @ s["k_pages"][page, hk, slot].double().t().contiguous() / math.sqrt(D)
            if case["causal"]:
                w = w.masked_fill(key.unsqueeze(0) > torch.arange(m - n, m, device="cuda").unsqueeze(1), float("-inf"))
            o[:, h] = torch.softmax(w, 1) @ s["v_pages"][page, hk, slot].double()
        put(o)
    return {"q": out, "k_pages": kc, "v_pages": vc} if kind == "append" else out
