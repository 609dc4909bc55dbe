"""Attention over a million places and more where one CTA, or one warp, has all of them: sums that stay exact over long stretches."""
import math

import pytest
import torch

from test_gpu_paged_attention import call, npu  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu
PAGE = 4096


def make_long(dev, places, heads, dim, dtype, batch, seed=0, distinct=16, rise=0.0):
    """One token of a sequence that names `distinct` pages again and again, its last page with scores that are higher by `rise`; the
    other sequences have one place."""
    g = torch.Generator(device=dev).manual_seed(seed)
    k = (torch.randn((distinct + 1, PAGE, 1, dim), generator=g, device=dev) * 0.5).to(dtype)
    v = (0.5 + torch.rand((distinct + 1, PAGE, 1, dim), generator=g, device=dev)).to(dtype)
    q = torch.randn((batch, heads, dim), generator=g, device=dev).to(dtype)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[distinct, :, 0, 0] = rise * math.sqrt(dim)
    columns = places // PAGE
    table = (torch.arange(columns, device=dev) % distinct).int().repeat(batch, 1)
    table[:, -1] = distinct
    lens = torch.ones(batch, dtype=torch.int32, device=dev)
    lens[0] = places
    return q, k, v, table, lens, torch.arange(batch + 1, dtype=torch.int32, device=dev)


def definition(q, k, v, table, row=0):
    """(out, lse) of a row in 64 bits, of a sequence that sees all that the table names: every page's keys as often as it does."""
    times = torch.bincount(table[0].long(), minlength=k.shape[0]).double().repeat_interleave(PAGE)
    x = q[row].double() @ k.view(-1, k.shape[-1]).double().t() * q.shape[2] ** -0.5
    lse = torch.logsumexp(x + times.log(), 1)
    p = torch.exp(x - lse[:, None]) * times
    return p @ v.view(-1, v.shape[-1]).double(), lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim,places,batch", [(1, 64, 1 << 20, 301), (1, 128, 1 << 20, 301), (160, 128, 1 << 20, 301), (7, 256, 1 << 20, 301),
                                                    (160, 80, 1 << 21, 301), (1, 128, (1 << 17) + PAGE, 301), (4, 128, 1 << 24, 1)])
@pytest.mark.parametrize("rise", [0.0, 9.0])
def test_long_sums(npu, dev, heads, dim, places, batch, dtype, rise):
    """A weight is rounded (u, by chance alike), the output as well; sums over stretches of 2^16 places (2^17 where a table is no longer)
    lose up to 2^-11, all towards 0; scores have sums of `dim` products in fp32 (2^-24 each of some 16)."""
    q, k, v, table, lens, starts = make_long(dev, places, heads, dim, dtype, batch, seed=dim + heads, rise=rise)
    out, lse = call(npu, q, k, v, table, lens, starts)
    want, want_lse = definition(q, k, v, table)
    u = torch.finfo(dtype).eps / 2
    assert ((out[0].double() / want - 1).abs().max().item()) <= 2 * u + 2.0 ** -11 + 2.0 ** -12
    assert (lse[0].double() - want_lse).abs().max().item() <= 2.0 ** -12
    if batch > 1:
        assert torch.equal(out[1:], v[table[1, 0].long(), 0].expand(batch - 1, heads, dim))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim", [(4, 64), (20, 128), (1, 256), (3, 72)])
@pytest.mark.parametrize("rise", [0.0, 9.0])
def test_long_sums_of_single_tokens(npu, dev, heads, dim, dtype, rise):
    """As above; 301 sequences of 2^21 places, some shorter, give a warp half a million places of one or of neighbours."""
    q, k, v, table, lens, _ = make_long(dev, 1 << 21, heads, dim, dtype, 301, seed=dim, rise=rise)
    lens[:] = 1 << 21
    lens[5:9] = torch.tensor([1, 3, 0, 1], device=dev)
    out, lse = call(npu, q, k, v, table, lens, None)
    u = torch.finfo(dtype).eps / 2
    for row in (0, 1, 4, 9, 77, 150, 300):
        want, want_lse = definition(q, k, v, table, row)
        assert ((out[row].double() / want - 1).abs().max().item()) <= 2 * u + 2.0 ** -11 + 2.0 ** -12
        assert (lse[row].double() - want_lse).abs().max().item() <= 2.0 ** -12
    assert torch.equal(out[5], v[table[5, 0].long(), 0].expand(heads, dim)) and not out[7].any() and bool((lse[7] == -math.inf).all())
    assert bool(out.isfinite().all())


def test_values_of_one_over_long_stretches_of_single_tokens(npu, dev):
    for heads, dim in ((4, 64), (20, 128), (1, 256)):
        q, k, v, table, lens, _ = make_long(dev, 1 << 21, heads, dim, torch.float16, 301, seed=9)
        v.fill_(1.0)
        lens[:] = 1 << 21
        out, _ = call(npu, q, k, v, table, lens, None)
        assert (out.double() - 1).abs().max().item() <= 2.0 ** -11 + 2.0 ** -11


def test_values_of_one_over_long_items(npu, dev):
    """2^20 places, values of 1, f16: the output is their weights' sum, rounded, over the weights' sum."""
    for heads in (1, 160):
        q, k, v, table, lens, starts = make_long(dev, 1 << 20, heads, 128, torch.float16, 301, seed=5)
        v.fill_(1.0)
        out, _ = call(npu, q, k, v, table, lens, starts)
        assert (out.double() - 1).abs().max().item() <= 2.0 ** -11 + 2.0 ** -11


def test_values_not_finite_in_long_items(npu, dev):
    """A NaN at the last place of a long sequence, which the second last token does not see."""
    q, k, v, table, lens, starts = make_long(dev, 1 << 18, 4, 128, torch.bfloat16, 301, seed=6)
    start = starts.clone()
    start[0], start[1:] = 0, starts[1:] + 1
    q = torch.cat([q[:1], q])
    clean = call(npu, q, k, v, table, lens, start)
    v[16, PAGE - 1, 0, 3] = math.nan
    out, lse = call(npu, q, k, v, table, lens, start)
    assert torch.equal(lse, clean[1]) and bool(out[1, :, 3].isnan().all())
    rest = out.clone()
    rest[1, :, 3] = clean[0][1, :, 3]
    # both of the sequence's rows are made again, in another order: two results that are off by up to 2u each
    assert bool(((rest.double() / clean[0].double() - 1).abs() <= 4 * 2.0 ** -8).all()) and torch.equal(rest[2:], clean[0][2:])


def test_calls_at_the_same_time(npu, dev):
    """Two streams, and graphs captured one after the other: each call's sums are put by in its own scratch."""
    states = [make_long(dev, 1 << 19, 160, 128, torch.bfloat16, 301, seed=s) for s in (7, 8)]
    for state in states:
        state[4][:40] = 1 << 19
    want = [call(npu, *s) for s in states]
    torch.cuda.synchronize()
    streams, graphs, got = [torch.cuda.Stream() for _ in states], [], []
    for s in states:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(call(npu, *s))
    for _ in range(3):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
