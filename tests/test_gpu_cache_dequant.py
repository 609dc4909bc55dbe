"""An int8 paged cache read back into pages of another type, bit for bit against its definition."""
import math
import random
import sys
from pathlib import Path

import pytest
import torch

from oracle import quant_cache_oracle as oracle

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"
LENS = [0, 1, 5, 16, 17, 100, -3, 129]


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


def make(dev, lens=LENS, kv=2, dim=64, page=16, rows=64, dtype=torch.bfloat16, seed=0, columns=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)

    def table_of(size):
        need = [max(0, -(-n // size)) for n in lens]
        ids = rng.sample(range(sum(need) + 3), sum(need) + 3)
        table = torch.full((len(lens), max(need + [columns])), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = ids.pop()
        return table.to(dev), sum(need) + 3

    (table, pages), (out_table, out_pages) = table_of(page), table_of(rows)
    codes = [torch.randint(-128, 128, (pages, page, kv, dim), generator=g, device=dev, dtype=torch.int8) for _ in range(2)]
    scales = [torch.exp(torch.randn((pages, kv, page), generator=g, device=dev)) for _ in range(2)]
    outs = [torch.randn((out_pages, rows, kv, dim), generator=g, device=dev).to(dtype) for _ in range(2)]
    return [*codes, *scales, table, torch.tensor(lens, dtype=torch.int32, device=dev), *outs, out_table]


def same(x, y):
    return torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


def check(npu, *args, first=None):
    want = oracle.read_back(*args, first=first)
    assert npu.npu_paged_cache_dequant(*args, first_places=first) is None
    assert same(args[6], want[0]) and same(args[7], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kv,dim", [(1, 1), (3, 7), (2, 8), (1, 24), (4, 80), (8, 128), (2, 256), (40, 64), (5, 12)])
def test_heads(npu, dev, kv, dim, dtype):
    check(npu, *make(dev, kv=kv, dim=dim, dtype=dtype, seed=dim))


@pytest.mark.parametrize("page,rows", [(1, 1), (16, 16), (5, 64), (64, 5), (24, 128), (7, 3), (512, 16)])
def test_page_sizes(npu, dev, page, rows):
    check(npu, *make(dev, page=page, rows=rows, seed=page))


def test_many_sequences(npu, dev):
    rng = random.Random(1)
    check(npu, *make(dev, [rng.choice([0, 1, rng.randrange(60)]) for _ in range(300)], dim=16, kv=1, seed=2))
    check(npu, *make(dev, [0] * 40 + [3000] + [0] * 40, dim=16, kv=1, seed=3))
    check(npu, *make(dev, [], seed=4, columns=2))


def test_first_places(npu, dev):
    """Read from a place on; first places behind the end, and negative ones."""
    for seed in range(3):
        args = make(dev, seed=5 + seed)
        first = torch.tensor([0, 1, 2, 15, -7, 63, 5, 200 if seed else 128], dtype=torch.int32, device=dev)
        check(npu, *args, first=first)
    check(npu, *make(dev, [40, 40], seed=9), first=torch.tensor([2**31 - 1, -2**31], dtype=torch.int32, device=dev))


def test_first_places_beyond_all_capacities(npu, dev):
    """Empty sequences of the largest first places, crossed on the way from the one before to the one behind."""
    args = make(dev, [3000, 100, 0, 3001, 50, 2999], kv=1, dim=16, seed=19)
    check(npu, *args, first=torch.tensor([0, 2**31 - 1, 2**31 - 2, 1, 2**31 - 1, 0], dtype=torch.int32, device=dev))
    args = make(dev, [3000, 100, 3001], kv=1, dim=16, seed=20)
    args[5] = torch.full_like(args[5], 2**31 - 1)
    check(npu, *args, first=torch.tensor([0, 2**31 - 1, 1], dtype=torch.int32, device=dev))


def test_tables(npu, dev):
    """Lengths beyond either table, entries that name no page in either."""
    args = make(dev, [200, 300, 100], seed=10)
    args[4][0, 3], args[4][1, 2], args[8][2, 0], args[8][1, 1] = -1, len(args[0]), 2**31 - 1, -2**31
    check(npu, *args)
    args = make(dev, [64, 64], seed=11)
    args[5] = torch.tensor([2**31 - 1, 70], dtype=torch.int32, device=dev)
    check(npu, *args)
    check(npu, *args[:4], args[4][:, :2].contiguous(), *args[5:])
    check(npu, *args[:8], args[8][:, :0].contiguous())
    check(npu, args[0][:0], args[1][:0], args[2][:0], args[3][:0], *args[4:])
    check(npu, *args[:6], args[6][:0], args[7][:0], args[8])


def test_shared_pages(npu, dev):
    """Sequences that begin with the same pages of the cache."""
    args = make(dev, [100, 100], seed=12)
    args[4][1, :4] = args[4][0, :4]
    check(npu, *args)


def test_values_that_are_not_finite(npu, dev):
    args = make(dev, [100], dtype=torch.float16, seed=13)
    args[2][args[4][0, 1], 0, 3], args[3][args[4][0, 2], 1, 3], args[2][args[4][0, 3], 1] = math.nan, math.inf, 1e6
    check(npu, *args)


def test_strides(npu, dev):
    args = make(dev, kv=4, seed=14)
    want = oracle.read_back(*args)
    k, v, ks, vs, table, lens, ko, vo, out_table = args
    layouts = [lambda x: x.transpose(1, 2).contiguous().transpose(1, 2), lambda x: torch.cat([x.new_zeros(4), x.reshape(-1)])[4:].view(x.shape),
               lambda x: torch.stack([x, x], 1)[:, 1]]
    for a in layouts:
        for b in layouts:
            outs = b(ko), b(vo)
            npu.npu_paged_cache_dequant(a(k), a(v), a(ks), b(vs), table.t().contiguous().t(), lens, *outs,
                                        torch.cat([out_table, out_table], 1)[:, : out_table.shape[1]])
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_far_offsets(npu, dev):
    """Caches and pages beyond 2^32 bytes."""
    args = make(dev, [100, 40], kv=1, dim=128, seed=15)
    want = oracle.read_back(*args)

    def at_the_end(x, pages):
        y = torch.empty((pages, *x.shape[1:]), dtype=x.dtype, device=dev)
        y[-len(x):] = x
        return y

    pages, rows = 2**21 + 2**18, 2**18 + 2**15
    n, m = len(args[0]), len(args[6])
    far = [at_the_end(x, pages) for x in args[:4]]
    outs = [at_the_end(x, rows) for x in args[6:8]]
    assert far[0].numel() > 2**32 and outs[0].numel() * 2 > 2**32
    move = lambda t, by: torch.where(t < 0, t, t + by)  # noqa: E731
    npu.npu_paged_cache_dequant(*far, move(args[4], pages - n), args[5], *outs, move(args[8], rows - m))
    assert torch.equal(outs[0][-m:], want[0]) and torch.equal(outs[1][-m:], want[1])


def test_graph_and_stream(npu, dev):
    args = make(dev, [50, 90], seed=16)
    npu.npu_paged_cache_dequant(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        npu.npu_paged_cache_dequant(*args)
    args[5].copy_(torch.tensor([33, 17], dtype=torch.int32))
    args[0].neg_()
    args[6].zero_()
    args[7].zero_()
    want = oracle.read_back(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(args[6], want[0]) and torch.equal(args[7], want[1])


def test_lazy_clones_keep_what_they_held(npu, dev):
    args = make(dev, [50], seed=17)
    held = [x.clone() for x in args[6:8]]
    clones = [torch._lazy_clone(x) for x in args[6:8]]
    check(npu, *args)
    assert all(torch.equal(x, y) for x, y in zip(clones, held))


def test_refusals(npu, dev):
    names = ["key_cache", "value_cache", "key_scale", "value_scale", "block_table", "seq_lens", "key_out", "value_out", "out_table"]
    args = dict(zip(names, make(dev, [5, 9], seed=18)))

    def refused(text, **kw):
        with pytest.raises(RuntimeError, match=text):
            npu.npu_paged_cache_dequant(**{**args, **kw})

    refused("quantized cache", key_cache=args["key_cache"].half())
    refused("same shape", value_cache=args["value_cache"][:-1])
    refused("float32", key_scale=args["key_scale"].half())
    refused("float32", value_scale=args["value_scale"].transpose(1, 2))
    refused("unsupported dtype", key_out=args["key_out"].int(), value_out=args["value_out"].int())
    refused("dtype of key_out", value_out=args["value_out"].half())
    refused("should hold 2 heads", key_out=args["key_out"][:, :, :1], value_out=args["value_out"][:, :, :1])
    refused("same address", value_out=args["key_out"])
    refused("should not overlap", key_out=args["key_out"][:1].expand_as(args["key_out"]))
    refused("int32", seq_lens=args["seq_lens"].long())
    refused("int32", block_table=args["block_table"][:1])
    refused("int32", out_table=args["out_table"].long())
    refused("int32", out_table=args["out_table"].cpu())
    refused("first_places", first_places=args["seq_lens"][:1])
    refused("first_places", first_places=args["seq_lens"].long())
    refused("dense", key_out=args["key_out"].transpose(2, 3).contiguous().transpose(2, 3))
