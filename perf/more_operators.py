"""An int8 paged key-value cache as measurable cases: the rotary step that fills it, attention over it, and its reading back.

The cache holds int8 values [pages, page size, heads, dim] and one fp32 scale for every row of them [pages, heads, page size]; a
row is quantized by its largest magnitude as it is written.  A case is a dict of plain values: the path (``op``), its head layout
and sizes.  ``prepare`` makes what a serving program holds before the call (activations, a filled cache, block tables, lengths),
``run`` makes one pass and returns what it computes: through the public operators of ``torch_npu`` where ``own`` is true, in
elementary torch operations where it is false (32 bits; the rotation of what is quantized and its quotients in 64, since a value
may lie next to the border of two steps).  ``exact`` is the definition in 64 bits.

Paths: ``step`` (a decode step: the new token of each sequence is turned, quantized and written, then attends to its cache),
``attend`` (the attention alone), ``chunk`` (new tokens of a ragged batch are turned, quantized and written, and the cached
sequences read back in the activations' type for the attention of prompts), ``read`` (the reading back alone).
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
        # the first steps of one conversation: latency alone
        {"name": "step_small", "op": "step", "B": 1, "lo": 200, "hi": 200, "H": 32, "KV": 8, "D": 128, "page": 16, "window": 0,
         "sinks": 0, "rotary": 128, "axes": 1, "mode": "half", "order": "blocked", "reach": 40000, "dtype": "bf16"},
        # a step of a full batch of ragged conversations, 70B-class heads
        {"name": "step_batch", "op": "step", "B": 64, "lo": 500, "hi": 8000, "H": 64, "KV": 8, "D": 128, "page": 16, "window": 0,
         "sinks": 0, "rotary": 128, "axes": 3, "mode": "half", "order": "cyclic", "reach": 130000, "dtype": "bf16"},
        # a few short chats of a small model: seven query heads a key head, pages that end inside tiles
        {"name": "attend_short", "op": "attend", "B": 5, "lo": 1, "hi": 60, "H": 28, "KV": 4, "D": 80, "page": 5, "window": 0,
         "sinks": 0, "dtype": "f16"},
        # one long document: few rows, a long axis
        {"name": "attend_long", "op": "attend", "B": 1, "lo": 131071, "hi": 131071, "H": 32, "KV": 8, "D": 128, "page": 64,
         "window": 0, "sinks": 0, "dtype": "f16"},
        # streaming conversations: a window and the first tokens, half precision, small heads
        {"name": "attend_window", "op": "attend", "B": 32, "lo": 1000, "hi": 30000, "H": 32, "KV": 4, "D": 64, "page": 32,
         "window": 4096, "sinks": 4, "dtype": "f16"},
        # large heads, two query heads a key head, pages of an odd size
        {"name": "attend_wide", "op": "attend", "B": 32, "lo": 500, "hi": 8000, "H": 8, "KV": 4, "D": 256, "page": 24, "window": 0,
         "sinks": 0, "dtype": "bf16"},
        # a short second message of a conversation: latency alone
        {"name": "chunk_small", "op": "chunk", "B": 1, "new_lo": 17, "new_hi": 17, "past_lo": 200, "past_hi": 200, "H": 32, "KV": 8,
         "D": 128, "page": 16, "rotary": 128, "axes": 1, "mode": "half", "order": "blocked", "reach": 40000, "dtype": "bf16"},
        # a whole video prompt in one chunk, with time, height and width
        {"name": "chunk_prompt", "op": "chunk", "B": 1, "new_lo": 8192, "new_hi": 8192, "past_lo": 0, "past_hi": 0, "H": 32, "KV": 8,
         "D": 128, "page": 16, "rotary": 128, "axes": 3, "mode": "half", "order": "cyclic", "reach": 100000, "dtype": "bf16"},
        # later chunks of ragged prompts in half precision, part of each head rotated, pairs side by side
        {"name": "chunk_ragged", "op": "chunk", "B": 6, "new_lo": 100, "new_hi": 2000, "past_lo": 30, "past_hi": 5000, "H": 32, "KV": 4,
         "D": 80, "page": 24, "rotary": 64, "axes": 2, "mode": "interleave", "order": "blocked", "reach": 4000, "dtype": "f16"},
        # one short conversation taken up again
        {"name": "read_small", "op": "read", "B": 1, "lo": 333, "hi": 333, "H": 32, "KV": 8, "D": 128, "page": 16, "dtype": "f16"},
        # a full batch of ragged conversations, for a prompt attention over all of them
        {"name": "read_batch", "op": "read", "B": 64, "lo": 500, "hi": 8000, "H": 64, "KV": 8, "D": 128, "page": 16, "dtype": "bf16"},
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
    op = rng.choice(["step", "attend", "attend", "chunk", "read"])
    KV = rng.choice([1, 2, 4, 8, 8])
    D = rng.choice([64, 80, 96, 128, 128, 128, 128, 256])
    c = {"op": op, "B": _log(rng, 1, 128), "H": KV * rng.choice([1, 2, 4, 4, 5, 7, 8, 16]), "KV": KV, "D": D,
         "page": rng.choice([16, 16, 32, 64, 128, 24, 5]), "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if op in ("step", "attend"):
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        c |= {"window": window, "sinks": rng.choice([0, 4, rng.randrange(1, 200)]) if window else 0}
    if op in ("step", "chunk"):
        c |= {"rotary": rng.choice([D, D, D, D // 2]), "axes": rng.choice([1, 1, 2, 3, 3]), "mode": rng.choice(["half", "half", "interleave"]),
              "order": rng.choice(["blocked", "cyclic"]), "reach": _log(rng, 100, 1000000)}
    if op == "chunk":
        new, past = _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 30000)])
        c |= {"new_lo": _log(rng, 1, new), "new_hi": new, "past_lo": rng.randrange(0, past + 1), "past_hi": past}
    else:
        hi = _log(rng, 1, 131072)
        c |= {"lo": _log(rng, 1, hi), "hi": hi}
    # a cache no larger than that of the largest listed batch, no more new tokens' rows than a long prompt's, no more work
    while (c["B"] * (c["new_hi"] + c["past_hi"] if op == "chunk" else c["hi"]) * KV * D > 64 * 8000 * 8 * 128
           or (op == "chunk" and c["B"] * c["new_hi"] * (c["H"] + 2 * KV) * D > 8192 * 48 * 128)
           or work(c)["bytes"] > work(listed()[-1])["bytes"]):
        if c["B"] > 1:
            c["B"] = (c["B"] + 1) // 2
        elif op == "chunk":
            c["new_hi"], c["past_hi"] = c["new_hi"] // 2 + 1, c["past_hi"] // 2
            c["new_lo"], c["past_lo"] = min(c["new_lo"], c["new_hi"]), min(c["past_lo"], c["past_hi"])
        else:
            c["hi"] = c["hi"] // 2 + 1
            c["lo"] = min(c["lo"], c["hi"])
    return c


def _sections(case):
    """Frequencies of each axis: the first has the rest of the equal shares' division."""
    n, a = case["rotary"] // 2, case["axes"]
    return [n - (a - 1) * (n // a)] + [n // a] * (a - 1)


def _lengths(case):
    """(new tokens, all tokens) of each sequence, in an order that the seed does not change."""
    B = case["B"]
    if case["op"] != "chunk":
        return [1] * B, _spread(B, case["lo"], case["hi"])
    new, past = _spread(B, case["new_lo"], case["new_hi"]), _spread(B, case["past_lo"], case["past_hi"])
    return new, [n + p for n, p in zip(new, past[::-1])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype, H, KV, D, page = _DTYPES[case["dtype"]], case["H"], case["KV"], case["D"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def tables(need, more):
        """Pages in a random order for `need[b]` pages of each sequence, -1 behind them, and how many there are."""
        pages = sum(need) + more
        ids = torch.randperm(pages, generator=g, device="cuda").int()
        at = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
        col, n = torch.arange(max(need), device="cuda"), torch.tensor(need, device="cuda")
        return torch.where(col < n[:, None], ids[(at[:, None] + col).clamp(max=pages - 1)], -1).int(), pages

    new, length = _lengths(case)
    order = list(range(case["B"]))
    rng.shuffle(order)
    new, length = [new[i] for i in order], [length[i] for i in order]
    table, pages = tables([-(-n // page) for n in length], 7)
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    T = start[-1] + (3 if case["op"] == "chunk" else 0)  # the tokens of a chunk are padded
    s = {"op": case["op"], "table": table, "lens": torch.tensor(length, device="cuda", dtype=torch.int32), "most": max(length),
         "window": case.get("window", 0), "sinks": case.get("sinks", 0)}
    for x in ("k", "v"):
        # rows of normal values, some tokens' larger than others', quantized by their largest magnitude
        rows = normal(pages, page, KV, D) * torch.exp(0.5 * normal(pages, page, KV, 1))
        top = rows.abs().amax(-1, keepdim=True).float()
        s[x + "_cache"] = (rows / (top / 127)).round().to(torch.int8)
        s[x + "_scale"] = (top / 127).squeeze(-1).transpose(1, 2).contiguous()
        del rows, top
    if case["op"] == "attend":
        s["q"] = normal(T, H, D)
    if case["op"] in ("step", "chunk"):
        qkv = normal(T, (H + 2 * KV) * D)  # the fused projection's output: its parts are strided views
        s |= {"sections": _sections(case), "mode": case["mode"], "order": case["order"], "q": qkv[:, :H * D].view(T, H, D),
              "k": qkv[:, H * D:(H + KV) * D].view(T, KV, D), "v": qkv[:, (H + KV) * D:].view(T, KV, D),
              "positions": torch.randint(0, case["reach"], (case["axes"], T), generator=g, device="cuda"),
              "inv_freq": (10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])).float().cuda()}
        if case["axes"] == 1:
            s["positions"] = s["positions"][0]
        seq = torch.tensor([b for b, n in enumerate(new) for _ in range(n)], device="cuda")
        place = torch.tensor([m - n + i for n, m in zip(new, length) for i in range(n)], device="cuda")
        slots = table[seq, place // page].long() * page + place % page
        s["slots"] = torch.cat([slots, torch.full((T - start[-1],), -1, device="cuda")])
    if case["op"] in ("chunk", "read"):
        # pages of the activations' type, of 64 places, in which the sequences are laid for the attention of prompts
        s["out_table"], n = tables([-(-n // 64) for n in length], 3)
        s["k_out"], s["v_out"] = torch.zeros((2, n, 64, KV, D), device="cuda", dtype=dtype)
    return s


def run(s):
    if own:
        npu, q = _npu(), s.get("q")
        cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        if s["op"] in ("step", "chunk"):
            q = npu.npu_rotary_axes_quant_cache(q, s["k"], s["v"], s["positions"], s["inv_freq"], *cache, s["slots"],
                                                sections=s["sections"], rotary_mode=s["mode"], axis_order=s["order"])
        if s["op"] in ("step", "attend"):
            out = npu.npu_paged_quant_attention(q, *cache, s["table"], s["lens"], window=s["window"], sinks=s["sinks"])
            return out if s["op"] == "attend" else (q, *cache[2:], *out)
        npu.npu_paged_cache_dequant(*cache, s["table"], s["lens"], s["k_out"], s["v_out"], s["out_table"])
        return (s["k_out"], s["v_out"]) if s["op"] == "read" else (q, *cache[2:], s["k_out"], s["v_out"])
    q = s.get("q")
    if s["op"] in ("step", "chunk"):
        q = _plain_write(s)
    if s["op"] in ("step", "attend"):
        out = _plain_attention(s, q)
        return out if s["op"] == "attend" else (q, s["k_scale"], s["v_scale"], *out)
    _plain_read(s)
    return (s["k_out"], s["v_out"]) if s["op"] == "read" else (q, s["k_scale"], s["v_scale"], s["k_out"], s["v_out"])


def _plain_rotary(s, x, bits):
    """Angles in 64 bits (positions reach far), the rotation in those of `bits`."""
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
    c, d = angle.cos().to(bits)[:, None], angle.sin().to(bits)[:, None]
    y = x.to(bits, copy=True)
    first, second = (slice(0, n), slice(n, 2 * n)) if s["mode"] == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., first].to(bits), x[..., second].to(bits)
    y[..., first], y[..., second] = a * c - b * d, b * c + a * d
    return y


def _plain_write(s):
    """Keys turned, both quantized row by row and written; the query turned."""
    page = s["k_cache"].shape[1]
    kept = s["slots"] >= 0
    # padding's rows are written to the place of a row that is written anyway, with its values
    at = torch.where(kept, s["slots"], s["slots"][0])
    for x, y in (("k", _plain_rotary(s, s["k"], torch.float64)), ("v", s["v"].double())):
        y = torch.where(kept[:, None, None], y, y[:1])
        scale = (y.abs().amax(-1) / 127).float()
        s[x + "_cache"].view(-1, *y.shape[1:])[at] = torch.where(scale[..., None] > 0, (y / scale.double()[..., None]).round(), 0.0).to(torch.int8)
        s[x + "_scale"][at // page, :, at % page] = scale
    return _plain_rotary(s, s["q"], torch.float32).to(s["q"].dtype)


def _plain_rows(s, x):
    """Rows [B, most, KV, D] of a cache as the fp32 values they stand for, and whether they are a sequence's."""
    page, KV, D = s["k_cache"].shape[1:]
    j = torch.arange(s["most"], device="cuda")
    at = s["table"].long()[:, j // page]
    here = (at >= 0) & (j < s["lens"][:, None])
    slot = at.clamp(min=0) * page + j % page
    scale = s[x + "_scale"].transpose(1, 2).reshape(-1, KV)[slot]
    return s[x + "_cache"].view(-1, KV, D)[slot].float() * scale[..., None], here


def _plain_read(s):
    rows = s["k_out"].shape[1]
    for x in ("k", "v"):
        y, here = _plain_rows(s, x)
        j = torch.arange(s["most"], device="cuda")
        slot = s["out_table"].long()[:, j // rows] * rows + j % rows
        s[x + "_out"].view(-1, *y.shape[2:])[slot[here]] = y[here].to(s["k_out"].dtype)


def _plain_attention(s, q):
    """All sequences at once, padded to the longest: the visible keys' softmax in 32 bits."""
    (k, here), (v, _) = _plain_rows(s, "k"), _plain_rows(s, "v")
    B, H, D = q.shape
    KV = k.shape[2]
    back = s["lens"][:, None] - 1 - torch.arange(s["most"], device="cuda")
    seen = here & (back >= 0)
    if s["window"]:
        seen &= (back < s["window"]) | (torch.arange(s["most"], device="cuda") < s["sinks"])
    score = q.float().view(B, KV, H // KV, D) @ k.permute(0, 2, 3, 1) / math.sqrt(D)
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True)
    y = e @ v.transpose(1, 2) / torch.where(total == 0, 1.0, total)
    return y.view(B, H, D).to(q.dtype), (top + total.log()).view(B, H)


def work(case):
    H, KV, D = case["H"], case["KV"], case["D"]
    new, length = _lengths(case)
    T, row = sum(new), 2 * D + 8  # bytes of a key and a value in the cache
    w = {"bytes": 0, "flops": 0}
    if case["op"] in ("step", "chunk"):
        w["bytes"] += 4 * T * H * D + T * KV * (4 * D + row) + 8 * T * (case["axes"] + 1)
        w["flops"] += 3 * T * (H + KV) * case["rotary"] + 4 * T * KV * D
    if case["op"] in ("step", "attend"):
        keys = sum(n if not case["window"] else min(n, case["sinks"] + case["window"]) for n in length)
        w["bytes"] += keys * KV * row + 2 * T * H * D * (1 if case["op"] == "step" else 2) + 4 * T * H
        w["flops"] += 4 * keys * H * D
    else:
        read = sum(length) - (T if case["op"] == "chunk" else 0)  # what was written just now need not be read
        w["bytes"] += read * KV * row + 4 * sum(length) * KV * D
        w["flops"] += 2 * sum(length) * KV * D
    return w


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    rows = {x: s[x + "_cache"].double() * s[x + "_scale"].transpose(1, 2).double()[..., None] for x in ("k", "v")}
    scales = {x: s[x + "_scale"].double() for x in ("k", "v")}
    q = s.get("q")
    if case["op"] in ("step", "chunk"):
        q = _exact_rotary(case, s, s["q"])
        slots = s["slots"][s["slots"] >= 0]
        for x, y in (("k", _exact_rotary(case, s, s["k"])), ("v", s["v"].double())):
            y = y[s["slots"] >= 0]
            scale = (torch.linalg.vector_norm(y, ord=math.inf, dim=-1) / 127).float().double()
            steps = torch.where(scale[..., None] > 0, torch.round(y / scale[..., None]), 0.0).clamp(-128, 127)
            rows[x].flatten(0, 1)[slots] = steps * scale[..., None]
            scales[x][slots // page, :, slots % page] = scale
    first = () if case["op"] in ("attend", "read") else (q, scales["k"], scales["v"])
    lens = s["lens"].tolist()
    if case["op"] in ("chunk", "read"):
        out = {x: s[x + "_out"].double() for x in ("k", "v")}
        for b, n in enumerate(lens):
            j = torch.arange(n, device="cuda")
            for x in ("k", "v"):
                out[x][s["out_table"][b].long()[j // 64], j % 64] = rows[x][s["table"][b].long()[j // page], j % page]
        return (*first, out["k"], out["v"])
    G = case["H"] // case["KV"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    if case["op"] == "step":
        q = q.to(s["q"].dtype)  # what the first operator gives the second
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        if case["window"]:
            j = j[(n - 1 - j < case["window"]) | (j < case["sinks"])]
        keys, values = (rows[x][s["table"][b].long()[j // page], j % page] for x in ("k", "v"))
        x = torch.einsum("kgd,nkd->kgn", q[b].double().view(case["KV"], G, -1), keys) * case["D"] ** -0.5
        lse[b] = torch.logsumexp(x, -1).flatten()
        out[b] = torch.einsum("kgn,nkd->kgd", torch.softmax(x, -1), values).flatten(0, 1)
    return (*first, out, lse)


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
