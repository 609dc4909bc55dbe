"""Rotary positions on several axes, and their form that writes a paged cache, against the definition in 64 bits."""
import sys
from pathlib import Path

import pytest
import torch

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


@pytest.fixture(scope="module")
def paged():
    from oracle import paged_oracle

    return paged_oracle


def make(dev, T, heads=8, kv=2, dim=64, pairs=None, axes=1, dtype=torch.bfloat16, reach=5000, seed=0, wide=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    pairs = dim // 2 if pairs is None else pairs
    qkv = torch.randn((T, (heads + 2 * kv) * dim), generator=g, device=dev).to(dtype)
    q, k, v = (x.view(T, x.shape[1] // dim, dim) for x in qkv.split([heads * dim, kv * dim, kv * dim], 1))
    positions = torch.randint(-reach // 8, reach, (axes, T), generator=g, device=dev)
    inv_freq = (10000.0 ** (-torch.arange(pairs, device=dev, dtype=torch.float64) / max(pairs, 1))).float()
    return q, k, v, positions if wide else positions.int(), inv_freq


def within(got, ref, x):
    """One rounding to the type (half a step of the result), and in fp32: the angle's 2^-25 half turns, sine and cosine (2^-23 with
    that), two products and a sum, each 2^-24 of terms up to |a| + |b| <= 2 max|x| of the row: 2^-20 of it covers them."""
    bound = torch.finfo(got.dtype).eps / 2 * ref.abs() + 2.0 ** -20 * x.double().abs().amax(-1, keepdim=True)
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"off by {(err / bound).max().item():.2f} times the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mode", ["half", "interleave"])
@pytest.mark.parametrize("dim,pairs", [(64, 32), (128, 64), (128, 32), (80, 40), (80, 16), (256, 128), (6, 3), (7, 2), (64, 31), (10, 0),
                                       (1, 0), (24, 6), (8, 4), (16, 8), (200, 96)])
def test_head_dimensions(npu, paged, dev, dim, pairs, mode, dtype):
    for T in (1, 37, 701):
        q, k, _, positions, inv_freq = make(dev, T, dim=dim, pairs=pairs, dtype=dtype, seed=dim)
        got = npu.npu_rotary_axes(q, k, positions, inv_freq, sections=[pairs], rotary_mode=mode)
        for x, y in zip((q, k), got):
            assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
            within(y, paged.rotary(x, positions, inv_freq, interleaved=mode == "interleave"), x)
            assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.parametrize("order", ["blocked", "cyclic"])
@pytest.mark.parametrize("sections", [[64], [32, 32], [16, 24, 24], [24, 20, 20], [64, 0, 0], [22, 21, 21], [16, 16, 16, 16], [40, 0, 24],
                                      [8] * 8, [34, 30]])
def test_axes(npu, paged, dev, sections, order):
    q, k, _, positions, inv_freq = make(dev, 50, dim=128, axes=len(sections), seed=len(sections))
    # axis 0 takes what the others leave, so its own count is no limit
    if order == "cyclic" and any(a and n and a + len(sections) * (n - 1) >= 64 for a, n in enumerate(sections)):
        with pytest.raises(RuntimeError, match="cyclic"):
            npu.npu_rotary_axes(q, k, positions, inv_freq, sections=sections, axis_order=order)
        return
    got = npu.npu_rotary_axes(q, k, positions, inv_freq, sections=sections, axis_order=order)
    for x, y in zip((q, k), got):
        within(y, paged.rotary(x, positions, inv_freq, sections, cyclic=order == "cyclic"), x)


@pytest.mark.parametrize("T,heads,kv", [(0, 4, 2), (1, 64, 8), (3, 1, 1), (2, 0, 3), (2, 5, 0), (300, 7, 7), (1025, 40, 8)])
def test_sizes(npu, paged, dev, T, heads, kv):
    q, k, _, positions, inv_freq = make(dev, T, heads, kv, dim=128, seed=T)
    for x, y in zip((q, k), npu.npu_rotary_axes(q, k, positions[0], inv_freq)):
        assert y.shape == x.shape
        if x.numel():
            within(y, paged.rotary(x, positions, inv_freq), x)


def test_far_positions(npu, paged, dev):
    """Positions of 2^24 and more: fp32 angles would be off by whole radians."""
    q, k, _, _, inv_freq = make(dev, 6, dim=64, dtype=torch.float32)
    positions = torch.tensor([2**24 + 1, 2**31 - 1, -2**31, 10**9 + 7, 12345, 0], device=dev)
    for at in (positions, positions.int()):
        # the half turns' product in 64 bits: off by up to 2^31 / pi * 2^-52 of them, less than 2^-20
        within(npu.npu_rotary_axes(q, k, at, inv_freq)[0], paged.rotary(q, at, inv_freq), q)
    assert torch.equal(npu.npu_rotary_axes(q, k, positions * 0, inv_freq)[0], q)


def test_strides(npu, paged, dev):
    """Heads in front of tokens, views that begin off the vectors, rows that are not dense, positions by column."""
    q, k, _, positions, inv_freq = make(dev, 33, dim=128, axes=3, seed=5)
    want = npu.npu_rotary_axes(q.contiguous(), k.contiguous(), positions, inv_freq, sections=[24, 20, 20])
    for f in (lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
              lambda x: torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape),
              lambda x: torch.cat([x, x], 2)[..., :128],
              lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
              lambda x: torch.cat([x, x[..., :1]], 2)[..., :128]):
        got = npu.npu_rotary_axes(f(q), f(k), positions.t().contiguous().t(), inv_freq, sections=[24, 20, 20])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def cached(npu, q, k, v, positions, inv_freq, k_cache, v_cache, slots, **kw):
    return npu.npu_rotary_axes_cache(q, k, v, positions, inv_freq, k_cache, v_cache, slots, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,pairs,page", [(128, 64, 16), (64, 16, 1), (80, 40, 24), (6, 3, 5), (256, 128, 64)])
@pytest.mark.parametrize("wide", [True, False])
def test_cache(npu, dev, dim, pairs, page, dtype, wide):
    """Bit for bit what npu_rotary_axes gives, at the tokens' places; the rest of the cache, and padding's, as it was."""
    T = 77
    q, k, v, positions, inv_freq = make(dev, T, dim=dim, pairs=pairs, axes=2, dtype=dtype, seed=dim, wide=wide)
    sections = [pairs - pairs // 2, pairs // 2]
    pages = T // page + 4
    g = torch.Generator(device=dev).manual_seed(1)
    slots = torch.randperm(pages * page, generator=g, device=dev)[:T]
    slots[5], slots[9], slots[10] = -1, pages * page, -2**31
    slots = slots if wide else slots.int()
    base = torch.randn((2, pages, page, 2, dim), device=dev).to(dtype)
    for layout in ("places", "heads", "offset"):
        kc, vc = base[0].clone(), base[1].clone()
        if layout == "heads":
            kc = kc.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "offset":
            vc = torch.cat([vc.new_zeros(1), vc.reshape(-1)])[1:].view(vc.shape)
        got = cached(npu, q, k, v, positions, inv_freq, kc, vc, slots, sections=sections)
        want = npu.npu_rotary_axes(q, k, positions, inv_freq, sections=sections)
        assert torch.equal(got, want[0])
        kw, vw = base[0].reshape(-1, 2, dim).clone(), base[1].reshape(-1, 2, dim).clone()
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                kw[s], vw[s] = want[1][t], v[t]
        assert torch.equal(kc.reshape(-1, 2, dim), kw) and torch.equal(vc.reshape(-1, 2, dim), vw)


def test_cache_beyond_32_bits(npu, dev):
    pages = 140000
    kc = torch.empty((pages, 16, 8, 128), dtype=torch.bfloat16, device=dev)
    q, k, v, positions, inv_freq = make(dev, 3, 16, 8, 128)
    slots = torch.tensor([pages * 16 - 1, 131073 * 16, 7], device=dev)
    want = npu.npu_rotary_axes(q, k, positions, inv_freq, sections=[64])[1]
    vc = torch.empty_like(kc)
    cached(npu, q, k, v, positions, inv_freq, kc, vc, slots, sections=[64])
    assert torch.equal(kc.view(-1, 8, 128)[slots], want) and torch.equal(vc.view(-1, 8, 128)[slots], v)


def test_graph_and_stream(npu, dev):
    q, k, v, positions, inv_freq = make(dev, 9, dim=128)
    kc, vc = torch.zeros((2, 4, 16, 2, 128), dtype=q.dtype, device=dev)
    slots = torch.arange(9, device=dev)
    cached(npu, q, k, v, positions, inv_freq, kc, vc, slots, sections=[64])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cached(npu, q, k, v, positions, inv_freq, kc, vc, slots, sections=[64])
    positions += 3
    slots += 20
    want = npu.npu_rotary_axes(q, k, positions, inv_freq, sections=[64])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want[0]) and torch.equal(kc.view(-1, 2, 128)[20:29], want[1]) and torch.equal(vc.view(-1, 2, 128)[20:29], v)


def test_refusals(npu, dev):
    q, k, v, positions, inv_freq = make(dev, 4, axes=2)
    kc, vc = torch.zeros((2, 4, 16, 2, 64), dtype=q.dtype, device=dev)
    slots = torch.arange(4, device=dev)

    def refused(text, *a, error=RuntimeError, **kw):
        with pytest.raises(error, match=text):
            (npu.npu_rotary_axes if len(a) == 4 else npu.npu_rotary_axes_cache)(*a, **kw)

    s = [16, 16]
    refused("unsupported dtype", q.int(), k.int(), positions, inv_freq, sections=s)
    refused("dtype of query", q, k.float(), positions, inv_freq, sections=s)
    refused("same tokens and dim", q, k[:3], positions, inv_freq, sections=s)
    refused("float32 vector", q, k, positions, inv_freq.double(), sections=s)
    refused("int32 or int64", q, k, positions.float(), inv_freq, sections=s)
    refused("hold 4 tokens", q, k, positions[:, :3], inv_freq, sections=s)
    refused("one entry for each", q, k, positions, inv_freq)
    refused("one entry for each", q, k, positions, inv_freq, sections=[32])
    refused("add up", q, k, positions, inv_freq, sections=[16, 15])
    refused("between 0 and", q, k, positions, inv_freq, sections=[33, -1])
    refused("between 1 and 8 axes", q, k, positions[:1].expand(9, 4), inv_freq, sections=[32] + [0] * 8)
    refused("more frequencies", q, k, positions[0], torch.ones(33, device=dev))
    refused("above 256", q.repeat(1, 1, 5), k.repeat(1, 1, 5), positions, inv_freq, sections=s)
    refused("'half' or 'interleave'", q, k, positions, inv_freq, sections=s, rotary_mode="other")
    refused("'blocked' or 'cyclic'", q, k, positions, inv_freq, sections=s, axis_order="other")
    refused("should be on", q, k, positions.cpu(), inv_freq, sections=s)
    refused("shape of key", q, k, v[:, :1], positions, inv_freq, kc, vc, slots, sections=s)
    refused("should hold 2 heads", q, k, v, positions, inv_freq, kc[:, :, :1], vc[:, :, :1], slots, sections=s)
    refused("same shape", q, k, v, positions, inv_freq, kc, vc[:2], slots, sections=s)
    refused("dtype of the query", q, k, v, positions, inv_freq, kc.float(), vc.float(), slots, sections=s)
    refused("int32 or int64", q, k, v, positions, inv_freq, kc, vc, slots.float(), sections=s)
    refused("should hold 4 tokens", q, k, v, positions, inv_freq, kc, vc, slots[:3], sections=s)
    refused("should be on", q, k, v, positions, inv_freq, kc, vc, slots.cpu(), sections=s)
    one = [c[:1].expand(4, -1, -1, -1) for c in (kc, vc)]
    refused("should not overlap", q, k, v, positions, inv_freq, *one, slots, sections=s)
