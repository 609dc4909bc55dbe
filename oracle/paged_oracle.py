"""Definitions in 64 bits of the operators over a paged key-value cache, for the tests."""
from __future__ import annotations

import math

import torch


def axis_of(i, sections, cyclic):
    if cyclic:
        a = i % len(sections)
        return a if i < len(sections) * sections[a] else 0
    for a, n in enumerate(sections):
        if i < n:
            return a
        i -= n
    raise AssertionError


def rotary(x, positions, inv_freq, sections=None, interleaved=False, cyclic=False):
    """x [T, H, D] turned, float64; positions [axes, T] or [T]."""
    n = inv_freq.numel()
    positions = positions.reshape(-1, x.shape[0])
    sections = sections or [n]
    axis = [axis_of(i, sections, cyclic) for i in range(n)]
    angle = positions[axis].double() * inv_freq.double()[:, None]
    c, s = angle.cos().t()[:, None], angle.sin().t()[:, None]
    y = x.double().clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def rows_of(lens, query_start, tokens):
    """(sequence, place) of each token, (-1, -1) for the tokens of no sequence."""
    if query_start is None:
        return [(b, n - 1) for b, n in enumerate(lens)]
    rows = [(-1, -1)] * tokens
    for b, n in enumerate(lens):
        for t in range(query_start[b], query_start[b + 1]):
            rows[t] = (b, n - (query_start[b + 1] - t))
    return rows


def seen(place, capacity, window, sinks):
    """Places that the token at `place` sees, bad pages aside."""
    return [j for j in range(min(place + 1, capacity)) if window == 0 or place - j < window or j < sinks]


def attention(q, k_cache, v_cache, table, lens, query_start=None, scale=None, window=0, sinks=0, only=None):
    """(out, lse, weight, spread, reach): the operator in float64 and, for bounds, sum_j p_j |v_j|, sum_j |v_j| and the largest sum_d |q_d k_jd| * scale
    of each row; places are gathered one row at a time.  only: the tokens that are computed."""
    T, H, D = q.shape
    pages, page, KV, _ = k_cache.shape
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros((T, H, D), dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    spread = torch.zeros_like(out)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros((T, H), dtype=torch.float64, device=q.device)
    rows = rows_of(lens.tolist(), None if query_start is None else query_start.tolist(), T)
    tables = table.tolist()
    for t, (b, place) in enumerate(rows):
        if b < 0 or (only is not None and t not in only):
            continue
        js = [j for j in seen(place, table.shape[1] * page, window, sinks) if 0 <= tables[b][j // page] < pages]
        if not js:
            continue
        js = torch.tensor(js, device=q.device)
        ids = table[b].long()[js // page]
        k = k_cache[ids, js % page].double().repeat_interleave(H // KV, 1)  # [n, H, D]
        v = v_cache[ids, js % page].double().repeat_interleave(H // KV, 1)
        x = torch.einsum("hd,nhd->hn", q[t].double(), k) * scale
        p = torch.softmax(x, 1)
        out[t] = torch.einsum("hn,nhd->hd", p, v)
        weight[t] = torch.einsum("hn,nhd->hd", p, v.abs())
        spread[t] = v.abs().sum(0)
        lse[t] = torch.logsumexp(x, 1)
        reach[t] = (torch.einsum("hd,nhd->hn", q[t].double().abs(), k.abs()) * abs(scale)).amax(1)
    return out, lse, weight, spread, reach


def attention_bounds(dtype, dim, out, lse, weight, spread, reach):
    """How far the operator's (out, lse) may be from the definition.

    u = half a step of the type.  A score is a sum of `dim` exact products in fp32 and two roundings more: off by at most
    d = (dim + 3) * 2^-24 * reach (reach: its terms' absolute sum).  A weight is exp of it (2^-21 covers exp2's own error, the
    rounding of the largest score and of the sums' rescaling), rounded to the type for the product with the values (u), so
        |out - ref| <= u |ref| + (u + 2 d + 2^-20) sum p |v|   and   |lse - ref| <= d + 2^-20 + 2^-22 |lse|.
    f16 has no full step below 2^-14: what lies there is off by up to 2^-25.  An output is as it is; weights are multiplied by
    2^11 at least, relative to a score that is 2^3 above the largest at most, so that the largest is 2^8 or more and the others
    are off by up to 2^-33 of it.
    """
    u = torch.finfo(dtype).eps / 2
    d = (dim + 3) * 2.0 ** -24 * reach
    bound = u * out.abs() + (u + 2 * d[..., None] + 2.0 ** -20) * weight
    if dtype == torch.float16:
        bound = bound + 2.0 ** -33 * spread + 2.0 ** -25
    return bound, d + 2.0 ** -20 + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)
