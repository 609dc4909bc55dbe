"""Attention over a paged key-value cache and the rotary step that fills it, as measurable cases.

A case is a dict of plain values: the operator (``op``), its head layout and sizes.  ``prepare`` makes what a serving program
holds before the call (activations, the cache's pages, block tables, lengths), ``run`` makes one pass and returns everything
that the operator returns or writes: through the public operators of ``torch_npu`` where ``own`` is true, in elementary torch
operations in 32 bits where it is false.  ``exact`` is the definition in 64 bits.

Operators: ``rotary`` (rotary positions on several axes), ``rotary_cache`` (the same, with the rotated keys and the values
written to their places in the paged cache), ``decode`` (attention of one new token a sequence), ``prompt`` (attention of the
new tokens of a ragged batch: whole prompts, later chunks of them, a few drafted tokens).  Both attentions read the paged
cache, whole or through a sliding window with a few first tokens that stay visible.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_PKG = str(Path(__file__).resolve().parent.parent / "ascend-python_b200")
_module = None


def _npu():
    global _module
    if _module is None:
        sys.path.insert(0, _PKG)
        try:
            import torch_npu
        finally:
            sys.path.remove(_PKG)
        _module = torch_npu
    return _module


def listed():
    return [
        # one image token or text token of each of four sequences: the smallest calls, where latency counts
        {"name": "rotary_small", "op": "rotary", "T": 4, "H": 32, "KV": 8, "D": 128, "rotary": 128, "axes": 3, "mode": "half",
         "order": "blocked", "reach": 40000, "dtype": "bf16"},
        # a video prompt: a whole prefill batch with time, height and width
        {"name": "rotary_video", "op": "rotary", "T": 8192, "H": 32, "KV": 8, "D": 128, "rotary": 128, "axes": 3, "mode": "half",
         "order": "cyclic", "reach": 100000, "dtype": "bf16"},
        # a decode step of 64 sequences, 70B-class heads: rotated keys and the values go to the cache
        {"name": "rotary_cache_decode", "op": "rotary_cache", "T": 64, "H": 64, "KV": 8, "D": 128, "rotary": 128, "axes": 1,
         "mode": "half", "order": "blocked", "reach": 130000, "page": 16, "spare": 64, "dtype": "bf16"},
        # a ragged prompt in half precision, part of each head rotated, pairs side by side
        {"name": "rotary_cache_ragged", "op": "rotary_cache", "T": 3001, "H": 32, "KV": 4, "D": 80, "rotary": 64, "axes": 2,
         "mode": "interleave", "order": "blocked", "reach": 4000, "page": 24, "spare": 9, "dtype": "f16"},
        # the first steps of one conversation: latency alone
        {"name": "decode_small", "op": "decode", "B": 1, "lo": 200, "hi": 200, "H": 32, "KV": 8, "D": 128, "page": 16,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # a full batch of ragged conversations, 70B-class heads
        {"name": "decode_batch", "op": "decode", "B": 64, "lo": 500, "hi": 8000, "H": 64, "KV": 8, "D": 128, "page": 16,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # one long document: few rows, a long axis
        {"name": "decode_long", "op": "decode", "B": 1, "lo": 131071, "hi": 131071, "H": 32, "KV": 8, "D": 128, "page": 64,
         "window": 0, "sinks": 0, "dtype": "bf16"},
        # streaming conversations: a window and the first tokens, half precision, small heads
        {"name": "decode_window", "op": "decode", "B": 32, "lo": 1000, "hi": 30000, "H": 32, "KV": 4, "D": 64, "page": 32,
         "window": 4096, "sinks": 4, "dtype": "f16"},
        # a short first message: latency alone
        {"name": "prompt_small", "op": "prompt", "B": 1, "new_lo": 17, "new_hi": 17, "past_lo": 0, "past_hi": 0, "H": 32, "KV": 8,
         "D": 128, "page": 16, "window": 0, "sinks": 0, "dtype": "bf16"},
        # a whole long prompt, 8B-class heads
        {"name": "prompt_long", "op": "prompt", "B": 1, "new_lo": 8192, "new_hi": 8192, "past_lo": 0, "past_hi": 0, "H": 32,
         "KV": 8, "D": 128, "page": 16, "window": 0, "sinks": 0, "dtype": "bf16"},
        # later chunks of prompts of several lengths, through a window with sinks
        {"name": "prompt_window", "op": "prompt", "B": 6, "new_lo": 100, "new_hi": 2000, "past_lo": 30, "past_hi": 5000, "H": 32,
         "KV": 8, "D": 128, "page": 32, "window": 1024, "sinks": 4, "dtype": "f16"},
        # a few drafted tokens of each of 16 sequences, checked against long caches: few rows, a long axis
        {"name": "prompt_draft", "op": "prompt", "B": 16, "new_lo": 3, "new_hi": 6, "past_lo": 2000, "past_hi": 16000, "H": 32,
         "KV": 8, "D": 128, "page": 16, "window": 0, "sinks": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """Uniform over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly spaced over their logarithm."""
    if n == 1:
        return [hi]
    lo_, hi_ = lo + 1.0, hi + 1.0
    return [int(round(lo_ * (hi_ / lo_) ** (i / (n - 1)))) - 1 for i in range(n)]


def draw(rng):
    op = rng.choice(["rotary", "rotary_cache", "decode", "decode", "prompt", "prompt"])
    KV = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    D = rng.choice([64, 80, 96, 128, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    page = rng.choice([16, 16, 32, 64, 128, 24, 5])
    if op in ("rotary", "rotary_cache"):
        rotary = rng.choice([D, D, D, D // 2])
        axes = rng.choice([1, 1, 2, 3, 3])
        c = {"op": op, "T": _log(rng, 1, 8192), "H": KV * group, "KV": KV, "D": D, "rotary": rotary, "axes": axes,
             "mode": rng.choice(["half", "half", "interleave"]), "order": rng.choice(["blocked", "cyclic"]),
             "reach": _log(rng, 100, 1000000), "dtype": dtype}
        if op == "rotary_cache":
            c |= {"page": page, "spare": rng.randrange(1, 64)}
        while c["T"] * (c["H"] + 2 * KV) * D > 8192 * 48 * 128:
            c["T"] = c["T"] // 2 + 1
        return c
    window = rng.choice([0, 0, _log(rng, 16, 8192)])
    sinks = rng.choice([0, 4, rng.randrange(1, 200)]) if window else 0
    c = {"op": op, "B": _log(rng, 1, 128), "H": KV * group, "KV": KV, "D": D, "page": page, "window": window, "sinks": sinks,
         "dtype": dtype}
    if op == "decode":
        hi = _log(rng, 1, 131072)
        c |= {"lo": _log(rng, 1, hi), "hi": hi}
        # the cache no larger than that of the largest listed batch
        while c["B"] * c["hi"] * KV * D > 64 * 8000 * 8 * 128:
            if c["B"] > 1:
                c["B"] = (c["B"] + 1) // 2
            else:
                c["hi"] = c["hi"] // 2 + 1
            c["lo"] = min(c["lo"], c["hi"])
        return c
    new, past = _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 30000)])
    c |= {"new_lo": _log(rng, 1, new), "new_hi": new, "past_lo": rng.randrange(0, past + 1), "past_hi": past}
    while (c["B"] * c["H"] * c["new_hi"] * (c["new_hi"] + c["past_hi"]) * max(D, 128) > 32 * 8192 * 8192 * 128
           or c["B"] * (c["new_hi"] + c["past_hi"]) * KV * D > 64 * 8000 * 8 * 128 or work(c)["flops"] > work(listed()[9])["flops"]):
        if c["B"] > 1:
            c["B"] = (c["B"] + 1) // 2
        else:
            c["new_hi"], c["past_hi"] = c["new_hi"] // 2 + 1, c["past_hi"] // 2
        c["new_lo"], c["past_lo"] = min(c["new_lo"], c["new_hi"]), min(c["past_lo"], c["past_hi"])
    return c


def _sections(case):
    """Frequencies of each axis: the first has the rest of the equal shares' division."""
    n, a = case["rotary"] // 2, case["axes"]
    return [n - (a - 1) * (n // a)] + [n // a] * (a - 1)


def _lengths(case):
    """(new tokens, all tokens) of each sequence, in an order that the seed does not change."""
    B = case["B"]
    if case["op"] == "decode":
        return [1] * B, _spread(B, case["lo"], case["hi"])
    new, past = _spread(B, case["new_lo"], case["new_hi"]), _spread(B, case["past_lo"], case["past_hi"])
    return new, [n + p for n, p in zip(new, past[::-1])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype, H, KV, D = _DTYPES[case["dtype"]], case["H"], case["KV"], case["D"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    if case["op"] in ("rotary", "rotary_cache"):
        T = case["T"]
        qkv = normal(T, (H + 2 * KV) * D)  # the fused projection's output: its parts are strided views
        s = {"op": case["op"], "sections": _sections(case), "mode": case["mode"], "order": case["order"],
             "q": qkv[:, :H * D].view(T, H, D), "k": qkv[:, H * D:(H + KV) * D].view(T, KV, D),
             "v": qkv[:, (H + KV) * D:].view(T, KV, D),
             "positions": torch.randint(0, case["reach"], (case["axes"], T), generator=g, device="cuda"),
             "inv_freq": (10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])).float().cuda()}
        if case["axes"] == 1:
            s["positions"] = s["positions"][0]
        if case["op"] == "rotary_cache":
            pages = -(-T // case["page"]) + case["spare"]
            s["k_cache"], s["v_cache"] = normal(pages, case["page"], KV, D), normal(pages, case["page"], KV, D)
            slots = torch.randperm(pages * case["page"], generator=g, device="cuda")[:T]
            s["slots"] = torch.where(torch.arange(T, device="cuda") % 61 == 60, -1, slots)  # a few rows of padding
        return s
    new, length = _lengths(case)
    order = list(range(case["B"]))
    rng.shuffle(order)
    new, length = [new[i] for i in order], [length[i] for i in order]
    page = case["page"]
    need = [-(-n // page) for n in length]
    pages = sum(need) + 7
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    at = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    col = torch.arange(max(need), device="cuda")
    need = torch.tensor(need, device="cuda")
    table = torch.where(col < need[:, None], ids[(at[:, None] + col).clamp(max=pages - 1)], -1).int()
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    return {"op": case["op"], "q": normal(start[-1], H, D), "k_cache": normal(pages, page, KV, D),
            "v_cache": normal(pages, page, KV, D), "table": table, "lens": torch.tensor(length, device="cuda", dtype=torch.int32),
            "start": torch.tensor(start, device="cuda", dtype=torch.int32), "window": case["window"], "sinks": case["sinks"],
            "most_new": max(new), "most": max(length)}


def run(s):
    if own:
        npu = _npu()
        if s["op"] == "rotary":
            return npu.npu_rotary_axes(s["q"], s["k"], s["positions"], s["inv_freq"], sections=s["sections"], rotary_mode=s["mode"],
                                       axis_order=s["order"])
        if s["op"] == "rotary_cache":
            q = npu.npu_rotary_axes_cache(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"],
                                          s["slots"], sections=s["sections"], rotary_mode=s["mode"], axis_order=s["order"])
            return q, s["k_cache"], s["v_cache"]
        if s["op"] == "decode":
            return npu.npu_paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], window=s["window"],
                                           sinks=s["sinks"])
        return npu.npu_paged_prompt_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["start"],
                                              window=s["window"], sinks=s["sinks"])
    if s["op"] == "rotary":
        return _plain_rotary(s, s["q"]), _plain_rotary(s, s["k"])
    if s["op"] == "rotary_cache":
        kept = s["slots"] >= 0
        k, v = s["k_cache"].view(-1, *s["k"].shape[1:]), s["v_cache"].view(-1, *s["v"].shape[1:])
        # padding's rows are written to the place of a row that is written anyway, with its values
        at = torch.where(kept, s["slots"], s["slots"][0])
        k[at] = torch.where(kept[:, None, None], _plain_rotary(s, s["k"]), _plain_rotary(s, s["k"])[:1])
        v[at] = torch.where(kept[:, None, None], s["v"], s["v"][:1])
        return _plain_rotary(s, s["q"]), s["k_cache"], s["v_cache"]
    return _plain_attention(s)


def _plain_rotary(s, x):
    """Angles in 64 bits (positions reach far), the rotation in 32 bits."""
    n = s["inv_freq"].numel()
    positions = s["positions"].view(-1, x.shape[0]).double()
    i = torch.arange(n, device="cuda")
    sections = torch.tensor(s["sections"], device="cuda")
    if s["order"] == "blocked":
        axis = (i[:, None] >= sections.cumsum(0)).sum(1)
    else:
        axis = i % len(s["sections"])
        axis = torch.where(i < len(s["sections"]) * sections[axis], axis, 0)
    angle = positions[axis].t() * s["inv_freq"].double()
    c, d = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.float().clone()
    if s["mode"] == "half":
        a, b = x[..., :n].float(), x[..., n:2 * n].float()
        y[..., :n], y[..., n:2 * n] = a * c - b * d, b * c + a * d
    else:
        a, b = x[..., 0:2 * n:2].float(), x[..., 1:2 * n:2].float()
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a * c - b * d, b * c + a * d
    return y.to(x.dtype)


def _plain_attention(s):
    """All sequences at once, padded to the longest: the visible keys' softmax in 32 bits."""
    q, kc, vc, table, lens, start = s["q"], s["k_cache"], s["v_cache"], s["table"].long(), s["lens"].long(), s["start"].long()
    T, H, D = q.shape
    page, KV = kc.shape[1], kc.shape[2]
    B, G = lens.numel(), H // KV
    j = torch.arange(s["most"], device="cuda")
    at = table[:, j // page]
    slot = at.clamp(min=0) * page + j % page
    k, v = kc.view(-1, KV, D)[slot].float().transpose(1, 2), vc.view(-1, KV, D)[slot].float().transpose(1, 2)
    i = torch.arange(s["most_new"], device="cuda")
    new = start[1:] - start[:-1]
    row = torch.where(i < new[:, None], start[:-1, None] + i, T)  # T: rows of padding
    pos = (lens - new)[:, None] + i
    back = pos[:, :, None] - j
    seen = (back >= 0) & (at >= 0)[:, None]
    if s["window"]:
        seen &= (back < s["window"]) | (j < s["sinks"])
    x = q[row.clamp(max=T - 1)].float().view(B, -1, KV, G, D).permute(0, 2, 1, 3, 4).reshape(B, KV, -1, D)
    score = (x @ k.transpose(2, 3) / math.sqrt(D)).view(B, KV, -1, G, s["most"])
    score = torch.where(seen[:, None, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    y = (e.view(B, KV, -1, s["most"]) @ v).view(B, KV, -1, G, D) / torch.where(total == 0, 1.0, total)
    out = torch.zeros((T + 1, H, D), device="cuda", dtype=q.dtype)
    lse = torch.full((T + 1, H), -math.inf, device="cuda")
    out[row] = y.permute(0, 2, 1, 3, 4).reshape(B, -1, H, D).to(q.dtype)
    lse[row] = (top + total.log()).squeeze(-1).permute(0, 2, 1, 3).reshape(B, -1, H)
    return out[:T], lse[:T]


def work(case):
    H, KV, D = case["H"], case["KV"], case["D"]
    if case["op"] in ("rotary", "rotary_cache"):
        heads = H + KV + (KV if case["op"] == "rotary_cache" else 0)
        return {"bytes": 4 * case["T"] * heads * D + 8 * case["T"] * (case["axes"] + (case["op"] == "rotary_cache")),
                "flops": 3 * case["T"] * (H + KV) * case["rotary"]}
    new, length = _lengths(case)
    pairs = sum(_pairs(case, n, a) for n, a in zip(new, length))
    keys = sum(a if not case["window"] else min(a, case["sinks"] + case["window"] + n - 1) for n, a in zip(new, length))
    return {"bytes": 4 * keys * KV * D + 4 * sum(new) * H * D + 4 * sum(new) * H, "flops": 4 * pairs * H * D}


def _pairs(case, n, length):
    """Visible (token, key) pairs of the last n tokens of `length`."""
    w, k = case["window"], case["sinks"]
    whole = n * length - n * (n - 1) // 2
    if not w:
        return whole
    # of token at place p (1-based length p), max(0, p - w - k) keys are neither in the window nor among the sinks
    hi, lo = max(0, length - w - k), max(0, length - n - w - k)
    return whole - (hi * (hi + 1) - lo * (lo + 1)) // 2


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rotary", "rotary_cache"):
        turned = {x: _exact_rotary(case, s, s[x]) for x in ("q", "k")}
        if case["op"] == "rotary":
            return turned["q"], turned["k"]
        k, v = s["k_cache"].double(), s["v_cache"].double()
        for t, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                k[slot // case["page"], slot % case["page"]] = turned["k"][t]
                v[slot // case["page"], slot % case["page"]] = s["v"][t].double()
        return turned["q"], k, v
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    G = case["H"] // case["KV"]
    starts, lens = s["start"].tolist(), s["lens"].tolist()
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        ids = s["table"][b, :-(-length // case["page"])].long()
        keys, values = s["k_cache"][ids].flatten(0, 1)[:length], s["v_cache"][ids].flatten(0, 1)[:length]
        where = torch.arange(length - n, length, device="cuda")[:, None] - torch.arange(length, device="cuda")
        hidden = where < 0
        if case["window"]:
            hidden |= (where >= case["window"]) & (torch.arange(length, device="cuda") >= case["sinks"])
        for h in range(case["H"]):
            x = s["q"][starts[b]:starts[b + 1], h].double() @ keys[:, h // G].double().t() * case["D"] ** -0.5
            x = x.masked_fill(hidden, -math.inf)
            lse[starts[b]:starts[b + 1], h] = torch.logsumexp(x, 1)
            out[starts[b]:starts[b + 1], h] = torch.softmax(x, 1) @ values[:, h // G].double()
    return out, lse


def _exact_rotary(case, s, x):
    """Pair by pair as complex numbers: the pair of frequency i turns by inv_freq[i] times the position on its axis."""
    n, sections = case["rotary"] // 2, s["sections"]
    if case["order"] == "blocked":
        axis = [a for a, m in enumerate(sections) for _ in range(m)]
    else:
        axis = [i % len(sections) if i < len(sections) * sections[i % len(sections)] else 0 for i in range(n)]
    p = s["positions"].reshape(case["axes"], -1).double()[axis]
    turn = torch.polar(torch.ones_like(p), p * s["inv_freq"].double()[:, None]).t()[:, None]
    y = x.double()
    first, second = (slice(0, n), slice(n, 2 * n)) if case["mode"] == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    z = torch.complex(y[..., first], y[..., second]) * turn
    y = y.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y
