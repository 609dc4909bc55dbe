"""Attention of one new token a sequence over an int8 paged cache against its definition in 64 bits."""
import math
import random
import sys
from pathlib import Path

import pytest
import torch

from oracle import quant_cache_oracle as oracle

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


def make(dev, lens, heads=8, kv=2, dim=64, page=16, dtype=torch.bfloat16, seed=0, spare=3, columns=0, size=1.0, key_size=0.02, spread=0.5):
    """Query, cache, scales, table and lengths.  Places behind a sequence's end have codes of any value and scales of NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    need = [max(0, -(-n // page)) for n in lens]
    pages = sum(need) + spare
    ids = list(range(pages))
    rng.shuffle(ids)
    table = torch.full((len(lens), max(need + [columns])), -1, dtype=torch.int32)
    k, v = (torch.randint(-128, 128, (pages, page, kv, dim), generator=g, device=dev, dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.full((pages, kv, page), math.nan, device=dev) for _ in range(2))
    for b, n in enumerate(lens):
        for i in range(need[b]):
            table[b, i] = ids.pop()
            rows = min(page, n - i * page)
            for s, by in ((ks, key_size), (vs, 0.02)):
                s[table[b, i], :, :rows] = by * torch.exp(spread * torch.randn((kv, rows), generator=g, device=dev))
    q = (torch.randn((len(lens), heads, dim), generator=g, device=dev) * size).to(dtype)
    return q, k, v, ks, vs, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)


def check(npu, q, k, v, ks, vs, table, lens, **kw):
    out, lse = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    assert lse.shape == q.shape[:2] and lse.dtype == torch.float32
    ref, ref_lse, bound, lse_bound = oracle.attention(q, k, v, ks, vs, table, lens, scale=kw.pop("scale_value", None), **kw)
    none = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, none) and bool((out[none] == 0).all())
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), f"out is off by {(err / bound).max().item():.2f} times its bound"
    err = (lse.double() - ref_lse)[~none].abs()
    assert bool((err <= lse_bound[~none]).all()), f"lse is off by {(err / lse_bound[~none]).max().item():.2f} times its bound"
    return out, lse


LENS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 100, 127, 128, 129, 255, 257, 300]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 112, 128, 144, 208, 256])
def test_head_dimensions(npu, dev, dim, dtype):
    check(npu, *make(dev, LENS, dim=dim, dtype=dtype, seed=dim))


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (7, 1), (12, 4), (16, 1), (34, 2), (32, 1), (40, 1)])
def test_groups(npu, dev, heads, kv):
    check(npu, *make(dev, LENS, heads=heads, kv=kv, dim=128, seed=heads))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 100, 128, 512])
def test_page_sizes(npu, dev, page, dim):
    check(npu, *make(dev, LENS, page=page, dim=dim, seed=page))


WINDOWS = [(1, 0), (1, 1), (7, 0), (16, 4), (33, 40), (64, 5), (100, 129), (128, 1), (1000, 4), (2**31, 2**31)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_window(npu, dev, window, sinks, dim):
    check(npu, *make(dev, LENS + [1000], dim=dim, seed=window % 97), window=window, sinks=sinks)


def test_long(npu, dev):
    """Split over the cache's length and joined; one sequence among short ones."""
    check(npu, *make(dev, [20011], heads=8, kv=2, dim=128, seed=1))
    check(npu, *make(dev, [3, 9000, 0, 40, 4097], heads=4, kv=4, dim=64, seed=2))
    check(npu, *make(dev, [5000, 77], heads=4, kv=2, dim=256, page=24, seed=3))
    check(npu, *make(dev, [700, 0, -5] * 40, heads=24, kv=2, dim=80, page=5, seed=4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-6])
def test_scales_of_scores(npu, dev, scale, dtype):
    check(npu, *make(dev, LENS, dim=128, dtype=dtype, seed=5), scale_value=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -8, 64.0, 2.0 ** 12])
def test_sizes_of_queries(npu, dev, size, dtype):
    """Rows of any magnitude: scores of the usual size by scales of the keys that make up for it."""
    check(npu, *make(dev, LENS, dim=128, dtype=dtype, seed=6, size=size, key_size=0.02 / size))


def test_query_elements_of_many_magnitudes(npu, dev):
    q, *rest = make(dev, LENS, dim=128, seed=7)
    q = (q.float() * 2.0 ** torch.linspace(-30, 3, 128, device=dev)).to(q.dtype)
    check(npu, q, *rest)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_peaked_scores(npu, dev, dtype):
    """Scores of hundreds: maxima that move far, weights of one key alone."""
    check(npu, *make(dev, LENS + [2000], dim=128, dtype=dtype, seed=8, size=30.0))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_value_scales_of_many_magnitudes(npu, dev, dim):
    """Values 2^40 apart: the weights' power of two follows the largest weight times scale of each row."""
    q, k, v, ks, vs, table, lens = make(dev, LENS + [3000], dim=dim, seed=9, size=4.0)
    vs = vs * 2.0 ** (torch.randint(-20, 21, vs.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(9)))
    check(npu, q, k, v, ks, vs, table, lens)
    vs = vs.nan_to_num(1.0) * 1e-30  # all of them small
    check(npu, q, k, v, ks, vs, table, lens)


def test_order_of_value_scales(npu, dev):
    """Ever larger values behind small ones and the other way round, equal scores."""
    for turn in (1.0, -1.0):
        q, k, v, ks, vs, table, lens = make(dev, [1024], dim=128, page=1024, heads=2, kv=2, spare=0, seed=10)
        vs[0] = 2.0 ** (turn * torch.linspace(-20, 20, 1024, device=dev))
        check(npu, q * 0, k, v, ks, vs, table, lens)
        check(npu, q, k, v, ks, vs, table, lens)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_far_above_those_before(npu, dev, dim):
    """A power of two that suits values of 2^-104 would take weights of values of 2^16 beyond fp32; and the other way round."""
    for small, large in ((range(0, 500), range(500, 900)), (range(500, 900), range(0, 500))):
        q, k, v, ks, vs, table, lens = make(dev, [900], dim=dim, page=1024, heads=2, kv=1, spare=0, seed=20, dtype=torch.bfloat16)
        vs[0, :, list(small)] = 2.0 ** -110
        vs[0, :, list(large)] = 2.0 ** 10
        # so many sequences, all of this page, that a CTA has whole ones
        check(npu, q.repeat(400, 1, 1), k, v, ks, vs, table.repeat(400, 1), lens.repeat(400))


def test_first_values_are_outweighed(npu, dev):
    """A key of a large value whose weight vanishes when the maximum moves; what counts lies 2^60 below it."""
    q, k, v, ks, vs, table, lens = make(dev, [300], dim=64, page=512, heads=1, kv=1, spare=0, seed=11)
    q[:], k[:] = 1.0, 1
    ks[0, 0, :300] = torch.linspace(0.01, 20.0, 300, device=dev)  # scores up to 160
    vs[0, 0, :300] = 1e-6
    vs[0, 0, :40] = 1e6
    check(npu, q, k, v, ks, vs, table, lens)


def test_zero_rows(npu, dev):
    """Scales of 0: keys that score 0, values that add nothing."""
    q, k, v, ks, vs, table, lens = make(dev, LENS, dim=128, seed=12)
    ks[:, :, ::3] = torch.where(ks[:, :, ::3].isnan(), math.nan, 0.0)
    vs[:, :, 1::2] = torch.where(vs[:, :, 1::2].isnan(), math.nan, 0.0)
    check(npu, q, k, v, ks, vs, table, lens)
    check(npu, q, k, v, ks, torch.where(vs.isnan(), vs, 0.0), table, lens)


def test_values_that_are_not_finite(npu, dev):
    """A row whose scale is NaN or infinite reaches the rows that see it, all of them, and no other."""
    for which in (0, 1):
        for bad in (math.nan, math.inf):
            q, k, v, ks, vs, table, lens = make(dev, [40, 70, 33], heads=8, kv=2, dim=64, seed=13)
            clean = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
            (ks, vs)[which][table[1, 2], 1, 5] = bad  # place 37 of sequence 1, head 1
            (k, v)[which][table[1, 2], 5, 1] = 0
            out, lse = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
            hit = torch.zeros(q.shape[:2], dtype=torch.bool, device=dev)
            hit[1, 4:] = True
            assert bool(out[hit].isnan().all()) and torch.equal(out[~hit], clean[0][~hit]) and torch.equal(lse[~hit], clean[1][~hit])
            if which == 0:
                assert bool(lse[hit].isnan().all())
            else:
                assert torch.equal(lse, clean[1])
            seen = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens, window=20)  # place 37 of 70 is behind
            assert bool(seen[0].isfinite().all())


def test_pages_that_are_none(npu, dev):
    """Table entries outside the cache, within a sequence: their places are not seen."""
    q, k, v, ks, vs, table, lens = make(dev, [100, 200, 16, 300], dim=128, seed=14)
    table[0, 2], table[1, 0], table[2, 0], table[3, 5] = -1, len(k), 2**31 - 1, -2**31
    out, lse = check(npu, q, k, v, ks, vs, table, lens)
    assert bool((lse[2] == -math.inf).all())


def test_lengths_beyond_the_table(npu, dev):
    q, k, v, ks, vs, table, _ = make(dev, [64, 64], dim=64, seed=15)
    check(npu, q, k, v, ks, vs, table, torch.tensor([70, 2**31 - 1], dtype=torch.int32, device=dev))
    check(npu, q, k, v, ks, vs, table[:, :0].contiguous(), torch.tensor([7, 0], dtype=torch.int32, device=dev))
    check(npu, q, k[:0], v[:0], ks[:0], vs[:0], table, torch.tensor([7, 0], dtype=torch.int32, device=dev))


def test_strides(npu, dev):
    """Heads in front of places, keys and values side by side, a query out of a projection, scales of any order, wide tables."""
    q, k, v, ks, vs, table, lens = make(dev, LENS, dim=64, kv=4, seed=16)
    want = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
    both = torch.stack([k, v], 3).transpose(1, 2).contiguous()  # [pages, heads, places, 2, dim]
    k2, v2 = both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2)
    scales = torch.stack([ks, vs], -1).permute(2, 0, 3, 1).contiguous()  # [places, pages, 2, heads]
    ks2, vs2 = scales[:, :, 0].permute(1, 2, 0), scales[:, :, 1].permute(1, 2, 0)
    q2 = torch.cat([q, q], 2).view(len(q), -1)[:, : 2 * q.shape[1] * 64].view(len(q), q.shape[1], 128)[:, :, :64]
    wide = torch.cat([table, torch.full_like(table, 7)], 1)[:, : table.shape[1]]
    got = npu.npu_paged_quant_attention(q2, k2, v2, ks2, vs2, wide, lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device=dev)[1:].view_as(q).copy_(q)
    got = npu.npu_paged_quant_attention(off, k, v, ks, vs, table.t().contiguous().t(), lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_far_offsets(npu, dev):
    """Caches of more than 2^32 bytes: pages at their end."""
    page, kv, dim, pages = 16, 1, 128, 2**21 + 2**18
    q, k, v, ks, vs, table, lens = make(dev, [100, 40], heads=4, kv=kv, dim=dim, page=page, seed=17)
    want = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)

    def at_the_end(x):
        y = torch.empty((pages, *x.shape[1:]), dtype=x.dtype, device=dev)
        y[-len(x):] = x
        return y

    far = [at_the_end(x) for x in (k, v, ks, vs)]
    assert far[0].numel() > 2**32
    got = npu.npu_paged_quant_attention(q, *far, torch.where(table < 0, table, table + (pages - len(k))), lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graphs_and_streams(npu, dev):
    """Captured and replayed with other contents; calls on another stream; the same bits every time."""
    q, k, v, ks, vs, table, lens = make(dev, [500, 3, 0, 2000], heads=16, kv=4, dim=128, seed=18)
    want = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    with torch.cuda.graph(graph):
        got = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
    lens2 = torch.tensor([17, 2000, 500, 1], dtype=torch.int32, device=dev)
    table2 = table[[0, 3, 0, 1]].contiguous()
    lens0, table0 = lens.clone(), table.clone()
    for l, t in ((lens2, table2), (lens0, table0)):
        lens.copy_(l)
        table.copy_(t)
        graph.replay()
        expect = npu.npu_paged_quant_attention(q, k, v, ks, vs, t, l)
        assert all(torch.equal(a, b) for a, b in zip(got, expect))
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens), want))


def test_refusals(npu, dev):
    q, k, v, ks, vs, table, lens = make(dev, [5, 9], dim=64, seed=19)
    good = dict(query=q, key_cache=k, value_cache=v, key_scale=ks, value_scale=vs, block_table=table, seq_lens=lens)
    for name, bad, text in (
            ("query", q.float(), "bfloat16 or float16"), ("query", q[:1], "one token"), ("query", q[:, :, :48].contiguous(), "head dimension"),
            ("query", q[:, :3].contiguous(), "multiple of the cache"), ("key_cache", k.half(), "quantized cache"), ("value_cache", v[:-1], "same shape"),
            ("value_cache", v.cpu(), "should be on"), ("key_scale", ks.half(), "float32"), ("value_scale", vs.transpose(1, 2), "float32"),
            ("key_scale", ks[:-1], "float32"), ("key_scale", ks.cpu(), "should be on"), ("block_table", table.long(), "int32"),
            ("seq_lens", lens[:1], "int32"), ("key_cache", k.transpose(2, 3), "dense")):
        with pytest.raises(RuntimeError, match=text):
            npu.npu_paged_quant_attention(**{**good, name: bad})
    for kw, text in ((dict(window=-1), "negative"), (dict(sinks=2), "window only"), (dict(scale_value=math.inf), "finite")):
        with pytest.raises(RuntimeError, match=text):
            npu.npu_paged_quant_attention(**good, **kw)
    odd = torch.zeros((4, 16, 2, 24), dtype=torch.int8, device=dev)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        npu.npu_paged_quant_attention(q[:, :, :24].contiguous(), odd, odd, ks[:4], vs[:4], table, lens)
    off = torch.zeros(k.numel() + 8, dtype=torch.int8, device=dev)[8:].view_as(k)
    with pytest.raises(RuntimeError, match="16-byte"):
        npu.npu_paged_quant_attention(q, off, v, ks, vs, table, lens)
