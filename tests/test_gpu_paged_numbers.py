"""Attention over the paged cache where its numbers can go wrong: one key that has nearly all the weight, runs of equal scores, values
that are not finite."""
import math

import pytest
import torch

from test_gpu_paged_attention import call, make, npu, paged  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def steps(dev, scores, dtype, heads=4, dim=64, page=64, new=None, batch=1):
    """Keys whose scores (scale 1) are `scores`, the same for every head; all sequences have the same pages."""
    n = scores.numel()
    pages = -(-n // page)
    k, v = torch.zeros((2, pages * page, 1, dim), dtype=dtype, device=dev)
    k[:n, 0, 0] = scores.to(dtype)
    table = torch.arange(pages, dtype=torch.int32, device=dev).repeat(batch, 1)
    q = torch.zeros((batch * (new or 1), heads, dim), dtype=dtype, device=dev)
    q[..., 0] = 1.0
    lens = torch.full((batch,), n, dtype=torch.int32, device=dev)
    starts = None if new is None else torch.arange(batch + 1, dtype=torch.int32, device=dev) * new
    return q, k.view(pages, page, 1, dim), v.view(pages, page, 1, dim), table, lens, starts


# (new tokens, sequences): one token, whose places all warps share; as many sequences as give a warp a long stretch; a prompt's
# token, whose places are split; as many as leave nothing to split
FORMS = [(None, 1), (None, 300), (1, 1), (1, 300)]


@pytest.mark.parametrize("new,batch", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("below", [13.0, 15.9, 16.3])
def test_one_key_with_nearly_all_the_weight(npu, dev, below, dtype, new, batch):
    """131071 keys far below the first, which has the value 0 where theirs is 1: their small weights are the whole output.

    A weight is rounded once (u relative, all alike), the output too; the sums are fp32, of at most 131072 terms in some 8192 steps of
    16 of one sign: 2^-24 each if every step rounds the same way, which is 2^-11.
    """
    n = 131072
    scores = torch.full((n,), -below, device=dev)
    scores[0] = 0.0
    q, k, v, table, lens, starts = steps(dev, scores, dtype, new=new, batch=batch)
    v[:] = 1.0
    v[0, 0] = 0.0
    out, lse = call(npu, q, k, v, table, lens, starts, scale_value=1.0)
    mass = (n - 1) * math.exp(float(k[0, 1, 0, 0]))
    want = mass / (1 + mass)
    u = torch.finfo(dtype).eps / 2
    assert (out.double() / want - 1).abs().max().item() <= 2 * u + 2.0 ** -11
    assert (lse.double() - math.log1p(mass)).abs().max().item() <= 2.0 ** -11


@pytest.mark.parametrize("new,batch", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rise", [0.3, 1.0, 2.7, 5.5])
def test_equal_scores_behind_lower_ones(npu, paged, dev, rise, dtype, new, batch):
    """Keys of one score behind a stretch of lower ones: where the base of the weights stays behind, all have the same weight,
    rounded the same way, while their sum is not rounded.  The bound has that rounding (u) beside the output's."""
    scores = torch.full((3000,), rise, device=dev)
    scores[:130] = 0.0
    q, k, v, table, lens, starts = steps(dev, scores, dtype, new=new, batch=batch)
    v.uniform_(0.9, 1.1, generator=torch.Generator(device=dev).manual_seed(3))
    out, lse = call(npu, q, k, v, table, lens, starts, scale_value=1.0)
    one = None if starts is None else starts[:2]
    ref = paged.attention(q[:1], k, v, table[:1], lens[:1], one, scale=1.0)
    bound, lse_bound = paged.attention_bounds(dtype, q.shape[2], *ref)
    assert bool(((out.double() - ref[0]).abs() <= bound).all()) and bool(((lse.double() - ref[1]).abs() <= lse_bound).all())


def same_as_definition(npu, paged, q, k, v, table, lens, starts, **kw):
    """Infinities and NaN as the definition has them, the rest within its bounds."""
    out, lse = call(npu, q, k, v, table, lens, starts, **kw)
    ref = paged.attention(q, k, v, table, lens, starts, **kw)
    bound, lse_bound = paged.attention_bounds(q.dtype, q.shape[2], *ref)
    odd = ~ref[0].isfinite()
    got = out.double()
    assert torch.equal(got[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), ref[0][odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
    assert bool(((got - ref[0]).abs() <= bound)[~odd].all())
    none = ref[1] == -math.inf
    assert torch.equal(lse == -math.inf, none) and bool(((lse.double() - ref[1]).abs() <= lse_bound)[~none].all())
    return odd


@pytest.mark.parametrize("window,sinks,page,dim", [(40, 4, 16, 128), (200, 4, 16, 128), (300, 20, 32, 256), (100, 3, 8, 64), (100, 4, 20, 128),
                                                   (0, 0, 16, 128), (1, 140, 64, 64)])
@pytest.mark.parametrize("split", [False, True])
def test_infinite_values(npu, paged, dev, window, sinks, page, dim, split):
    """A value that is infinite makes the rows that see it infinite, not NaN, whatever comes beside it in a tile; two of both signs NaN."""
    lens, new = ([3000, 1500], [6, 5]) if split else ([900, 700], [300, 260])
    for tokens in (None, new):
        q, k, v, table, length, starts = make(dev, lens, tokens, heads=4, kv=2, dim=dim, page=page, seed=dim + page)
        hit = 0
        for places in ((1,), (130,), (lens[0] - 3,), (2, lens[0] - 2)):
            for sign in (1.0, -1.0):
                v2 = v.clone()
                for i, j in enumerate(places):
                    v2[table[0, j // page], j % page, 1, 3] = math.inf * sign * (-1) ** i
                hit += int(same_as_definition(npu, paged, q, k, v2, table, length, starts, window=window, sinks=sinks).sum())
        assert hit > 0
