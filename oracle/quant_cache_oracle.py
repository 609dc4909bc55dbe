"""Definitions in 64 bits of the operators over an int8 paged key-value cache, for the tests."""
from __future__ import annotations

import torch

from oracle import paged_oracle


def quantize(y):
    """Codes (int8) and fp32 scales of rows y [..., dim] in float64."""
    top = torch.where(y.isnan().any(-1), torch.nan, y.abs().amax(-1)) if y.shape[-1] else y.new_zeros(y.shape[:-1])
    scale = (top / 127).float()
    fine = (scale > 0) & scale.isfinite()
    steps = y / torch.where(fine, scale, 1.0).double()[..., None]
    return torch.where(fine[..., None], steps, 0.0).round().clamp(-128, 127).to(torch.int8), scale


def values(codes, scale):
    """What codes [pages, page, heads, dim] and scales [pages, heads, page] stand for, float64."""
    return codes.double() * scale.double().transpose(1, 2)[..., None]


def attention(q, k_codes, v_codes, k_scale, v_scale, table, lens, scale=None, window=0, sinks=0):
    """(out, lse, out's bound, lse's bound) of one new token a sequence.

    As paged_oracle.attention_bounds, but for the weights and the query.  d: a query's element is a whole number, of a step of at most 2^-21
    of its row's largest, off by half a step, 2^-22 of that one.  A score's sum of products with codes is exact, but for its parts'
    roundings, and then multiplied by the key's scale, the row's power of two and scale_value: (dim + 5) * 2^-24 of its terms' absolute sum is more.  A weight, exp times the value's scale, is rounded to r of it, or
    half of f16's smallest step, 2^-25, where the row's largest weight is 2^8 or more: 2^-33 of that; r is half a step of f16, 2^-11, and for an f16 query, where a weight is the sum of two f16 numbers, 2^-22.
    So with w_j = p_j * value scale

        |out - ref| <= u |ref| + (r + 2 d + 2^-20) sum p |v| + 2^-33 max w sum |code|,   |lse - ref| <= d + 2^-20 + 2^-22 |lse|,

    whatever the number of places: a lane's weights of a tile are up to 8, what adding them to those before rounds away is kept, and that of the lanes, warps and
    parts is within 2^-20, too; u half a step of the output's type, and half of its smallest step more for an output below its full steps (f16 2^-25, bf16 2^-134).
    """
    k, v = values(k_codes, k_scale), values(v_codes, v_scale)
    out, lse, weight, _, reach = paged_oracle.attention(q, k, v, table, lens, scale=scale, window=window, sinks=sinks)
    T, H, D = q.shape
    pages, page, KV, _ = k_codes.shape
    by = D ** -0.5 if scale is None else scale
    spread = torch.zeros_like(out)
    most = torch.zeros_like(lse)
    far = torch.zeros_like(lse)  # the largest |q| times a key's sum of magnitudes
    tables = table.tolist()
    for t, n in enumerate(lens.tolist()):
        js = [j for j in paged_oracle.seen(n - 1, table.shape[1] * page, window, sinks) if 0 <= tables[t][j // page] < pages]
        if not js:
            continue
        js = torch.tensor(js, device=q.device)
        ids = table[t].long()[js // page]
        keys = k[ids, js % page].repeat_interleave(H // KV, 1)
        x = torch.einsum("hd,nhd->hn", q[t].double(), keys) * by
        p = torch.exp(x - lse[t][:, None])
        spread[t] = v_codes[ids, js % page].double().abs().sum(0).repeat_interleave(H // KV, 0)
        most[t] = (p * v_scale[ids, :, js % page].double().abs().t().repeat_interleave(H // KV, 0)).amax(1)
        far[t] = (keys.abs().sum(2).t() * abs(by)).amax(1) * q[t].double().abs().amax(1)
    d = (D + 5) * 2.0 ** -24 * reach + 2.0 ** -22 * far
    r = 2.0 ** -22 if q.dtype == torch.float16 else 2.0 ** -11
    bound = torch.finfo(q.dtype).eps / 2 * out.abs() + (r + 2 * d[..., None] + 2.0 ** -20) * weight + 2.0 ** -33 * most[..., None] * spread
    bound = bound + torch.finfo(q.dtype).smallest_normal * (torch.finfo(q.dtype).eps / 2)
    return out, lse, bound, d + 2.0 ** -20 + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)


def read_back(k_codes, v_codes, k_scale, v_scale, table, lens, k_out, v_out, out_table, first=None):
    """Copies of k_out and v_out with what the operator writes: the fp32 product, rounded once more to their type."""
    pages, page = k_codes.shape[:2]
    out_pages, rows = k_out.shape[:2]
    done = []
    for codes, scale, out in ((k_codes, k_scale, k_out.clone()), (v_codes, v_scale, v_out.clone())):
        for b, n in enumerate(lens.tolist()):
            for j in range(max(0, 0 if first is None else int(first[b])), min(n, table.shape[1] * page, out_table.shape[1] * rows)):
                at, to = int(table[b, j // page]), int(out_table[b, j // rows])
                if 0 <= at < pages and 0 <= to < out_pages:
                    out[to, j % rows] = (codes[at, j % page].float() * scale[at, :, j % page, None]).to(out.dtype)
        done.append(out)
    return tuple(done)
