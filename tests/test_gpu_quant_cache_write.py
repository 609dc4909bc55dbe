"""Rotary positions with the write into an int8 paged cache, code for code against the definition in 64 bits."""
import math
import sys
from pathlib import Path

import pytest
import torch

from oracle import paged_oracle
from oracle import quant_cache_oracle as oracle

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


def make(dev, T, heads=8, kv=2, dim=64, pairs=None, axes=1, dtype=torch.bfloat16, reach=5000, seed=0, page=16, spare=3):
    """(arguments of the operator, without options): the cache holds other codes and scales, some tokens go nowhere."""
    g = torch.Generator(device=dev).manual_seed(seed)
    pairs = dim // 2 if pairs is None else pairs
    qkv = torch.randn((T, (heads + 2 * kv) * dim), generator=g, device=dev).to(dtype)
    q, k, v = (x.view(T, x.shape[1] // dim, dim) for x in qkv.split([heads * dim, kv * dim, kv * dim], 1))
    positions = torch.randint(-reach // 8, reach, (axes, T), generator=g, device=dev)
    inv_freq = (10000.0 ** (-torch.arange(pairs, device=dev, dtype=torch.float64) / max(pairs, 1))).float()
    pages = -(-T // page) + spare
    slots = torch.randperm(pages * page, generator=g, device=dev)[:T]
    slots[5::19], slots[9::23] = -1, pages * page
    codes = [torch.randint(-128, 128, (pages, page, kv, dim), generator=g, device=dev, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand((pages, kv, page), generator=g, device=dev) for _ in range(2)]
    return [q, k, v, positions, inv_freq, *codes, *scales, slots]


def check(npu, q, k, v, positions, inv_freq, kc, vc, ks, vs, slots, sections=None, rotary_mode="half", axis_order="blocked"):
    sections = sections or [inv_freq.numel()]
    pages, page, kv, dim = kc.shape
    want = []
    turned = paged_oracle.rotary(k, positions, inv_freq, sections, rotary_mode == "interleave", axis_order == "cyclic") if len(k) else k.double()
    for y, codes, scales in ((turned, kc, ks), (v.double(), vc, vs)):
        new_codes, new_scales = oracle.quantize(y)
        codes, scales = codes.clone(), scales.clone()
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                codes[slot // page, slot % page], scales[slot // page, :, slot % page] = new_codes[t], new_scales[t]
        want.append((codes, scales))
    options = dict(sections=sections, rotary_mode=rotary_mode, axis_order=axis_order)
    out = npu.npu_rotary_axes_quant_cache(q, k, v, positions, inv_freq, kc, vc, ks, vs, slots, **options)
    assert torch.equal(out, npu.npu_rotary_axes(q, k, positions, inv_freq, **options)[0]) and out.is_contiguous()
    for (codes, scales), got_codes, got_scales in zip(want, (kc, vc), (ks, vs)):
        assert torch.equal(got_codes, codes)
        assert torch.equal(got_scales.isnan(), scales.isnan()) and torch.equal(got_scales.nan_to_num(7.0), scales.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mode", ["half", "interleave"])
@pytest.mark.parametrize("dim,pairs", [(64, 32), (128, 64), (128, 32), (80, 40), (80, 16), (256, 128), (6, 3), (7, 2), (64, 31), (10, 0),
                                       (1, 0), (24, 6), (8, 4), (16, 8), (200, 96), (136, 64), (256, 0)])
def test_head_dimensions(npu, dev, dim, pairs, mode, dtype):
    for T in (1, 37, 701):
        check(npu, *make(dev, T, dim=dim, pairs=pairs, dtype=dtype, seed=dim), rotary_mode=mode)


@pytest.mark.parametrize("order", ["blocked", "cyclic"])
@pytest.mark.parametrize("sections", [[32, 32], [24, 20, 20], [64, 0, 0], [8] * 8])
def test_axes(npu, dev, sections, order):
    if order == "cyclic" and sections == [24, 20, 20]:
        sections = [22, 21, 21]
    check(npu, *make(dev, 50, dim=128, axes=len(sections), seed=len(sections)), sections=sections, axis_order=order)


@pytest.mark.parametrize("T,heads,kv,page", [(0, 4, 2, 16), (1, 64, 8, 16), (3, 1, 1, 1), (2, 0, 3, 5), (300, 7, 7, 24), (1025, 40, 8, 128), (2100, 3, 1, 16)])
def test_sizes(npu, dev, T, heads, kv, page):
    check(npu, *make(dev, T, heads, kv, dim=128, seed=T, page=page))


def test_far_positions(npu, dev):
    """Positions whose fp32 angles would be off by whole radians."""
    args = make(dev, 6, dim=64, dtype=torch.float32)
    args[3] = torch.tensor([2**24 + 1, 2**31 - 1, -2**31, 10**9 + 7, 12345, 0], device=dev)
    args[9] = torch.arange(6, device=dev)
    check(npu, *args)
    args[3] = args[3].int()
    args[9] = args[9].int()
    check(npu, *args)
    args = make(dev, 900, dim=128, kv=8, reach=10**6, seed=3)
    check(npu, *args)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_and_special_rows(npu, dev, dtype):
    """Quotients of exactly a half and a half; rows of zeros, of the smallest numbers, with NaN and infinities."""
    T, dim = 12, 64
    args = make(dev, T, heads=1, kv=1, dim=dim, dtype=dtype, seed=4)
    args[3] = torch.zeros_like(args[3])
    args[9] = torch.arange(T, device=dev)
    y = torch.arange(dim, device=dev, dtype=torch.float64) - 31.5  # ties of a scale of 1
    y[0] = 127.0
    rows = torch.stack([y, -y, y * 2.0 ** -10, torch.zeros_like(y), y * 3, y.sign(), torch.full_like(y, torch.finfo(dtype).tiny),
                        y * float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps, torch.full_like(y, torch.finfo(dtype).max), y, y, y])
    rows = rows.to(dtype)
    rows[9, 5], rows[10, 7], rows[11, 2], rows[11, 3] = math.nan, math.inf, -math.inf, math.nan
    for turned in (rows[:, None], rows[:, None].flip(0)):
        args[1], args[2] = turned.contiguous(), turned.flip(2).contiguous()
        check(npu, *args)
    args[4] = args[4][:0]
    check(npu, *args)


def test_strides(npu, dev):
    """Heads in front of places or scales behind them, views that begin off the vectors, rows that are not dense."""
    for layout in ("heads", "offset", "together"):
        args = make(dev, 333, dim=128, kv=4, axes=3, seed=5)
        q, k, v, positions, inv_freq, kc, vc, ks, vs, slots = args
        if layout == "heads":
            kc, vc = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))
            ks, vs = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (ks, vs))
            k = k.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "offset":
            kc, vc = (torch.cat([x.new_zeros(n), x.reshape(-1)])[n:].view(x.shape) for x, n in ((kc, 8), (vc, 4)))
            q, v = (torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape) for x in (q, v))
        else:
            both = torch.stack([kc, vc], 1)
            kc, vc = both[:, 0], both[:, 1]
            both = torch.stack([ks, vs], 1)
            ks, vs = both[:, 0], both[:, 1]
        check(npu, q, k, v, positions.t().contiguous().t(), inv_freq, kc, vc, ks, vs, slots, sections=[24, 20, 20])


def test_beyond_32_bits(npu, dev):
    args = make(dev, 3, 16, 8, 128)
    pages = 280000
    kc, vc = (torch.empty((pages, 16, 8, 128), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.empty((pages, 8, 16), device=dev) for _ in range(2))
    slots = torch.tensor([pages * 16 - 1, 262145 * 16, 7], device=dev)
    npu.npu_rotary_axes_quant_cache(*args[:5], kc, vc, ks, vs, slots, sections=[64])
    turned = paged_oracle.rotary(args[1], args[3], args[4])
    for y, codes, scales in ((turned, kc, ks), (args[2].double(), vc, vs)):
        want = oracle.quantize(y)
        assert torch.equal(codes.view(-1, 8, 128)[slots], want[0]) and torch.equal(scales[slots // 16, :, slots % 16], want[1])


def test_graph_and_stream(npu, dev):
    q, k, v, positions, inv_freq, kc, vc, ks, vs, _ = make(dev, 9, dim=128, page=16)
    kc, vc, ks, vs = (x.repeat(4, *[1] * (x.dim() - 1)) for x in (kc, vc, ks, vs))
    slots = torch.arange(9, device=dev)
    npu.npu_rotary_axes_quant_cache(q, k, v, positions, inv_freq, kc, vc, ks, vs, slots, sections=[64])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = npu.npu_rotary_axes_quant_cache(q, k, v, positions, inv_freq, kc, vc, ks, vs, slots, sections=[64])
    positions += 3
    slots += 20
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, npu.npu_rotary_axes(q, k, positions, inv_freq, sections=[64])[0])
    codes, scale = oracle.quantize(paged_oracle.rotary(k, positions, inv_freq))
    assert torch.equal(kc.view(-1, 2, 128)[20:29], codes) and torch.equal(ks[slots // 16, :, slots % 16], scale)


def test_lazy_clones_keep_what_they_held(npu, dev):
    """A cache that shares its storage with a lazy clone is given its own before it is written, scales too."""
    args = make(dev, 20, dim=64)
    held = [x.clone() for x in args[5:9]]
    clones = [torch._lazy_clone(x) for x in args[5:9]]
    npu.npu_rotary_axes_quant_cache(*args, sections=[32])
    assert all(torch.equal(x, y) for x, y in zip(clones, held))
    assert not torch.equal(args[5], held[0])


def test_refusals(npu, dev):
    args = make(dev, 4, axes=2)

    def refused(text, **kw):
        names = ["query", "key", "value", "positions", "inv_freq", "key_cache", "value_cache", "key_scale", "value_scale", "slots"]
        with pytest.raises(RuntimeError, match=text):
            npu.npu_rotary_axes_quant_cache(**{**dict(zip(names, args)), "sections": [16, 16], **kw})

    q, k, v, positions, inv_freq, kc, vc, ks, vs, slots = args
    refused("unsupported dtype", query=q.int(), key=k.int())
    refused("dtype of query", key=k.float())
    refused("shape of key", value=v[:, :1])
    refused("add up", sections=[16, 15])
    refused("quantized cache", key_cache=kc.to(q.dtype))
    refused("same shape", value_cache=vc[:2])
    refused("should hold 2 heads", key_cache=kc[:, :, :1], value_cache=vc[:, :, :1], key_scale=ks[:, :1], value_scale=vs[:, :1])
    refused("float32", key_scale=ks.double())
    refused("float32", value_scale=vs[:, :, :-1])
    refused("should be on", value_scale=vs.cpu())
    refused("should be on", slots=slots.cpu())
    refused("int32 or int64", slots=slots.float())
    refused("should hold 4 tokens", slots=slots[:3])
    refused("should not overlap", key_cache=kc[:1].expand_as(kc))
    refused("should not overlap", value_scale=vs[:, :, :1].expand_as(vs))
    refused("same address", value_cache=kc)
    refused("same address", value_scale=ks)
