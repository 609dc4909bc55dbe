"""The operators of a quantized decoder layer with an int8 cache in a row, as a server runs them: normalisation and quantization, the
fused QKV projection, rotary positions with the cache write, for prompts the cache read back and attention over its pages, for single
tokens attention over the cache itself, quantization, the output projection."""
import sys
from pathlib import Path

import pytest
import torch

from oracle import paged_oracle
from oracle import quant_cache_oracle as oracle

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"
HEADS, KV, DIM, HIDDEN, PAGE, ROWS = 16, 4, 128, 1024, 16, 64


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


class Layer:
    def __init__(self, npu, dev, dtype, pages):
        g = torch.Generator(device=dev).manual_seed(1)
        self.npu, self.dtype, self.dev = npu, dtype, dev
        self.gamma = (1 + 0.1 * torch.randn(HIDDEN, generator=g, device=dev)).to(dtype)
        self.qkv = torch.randint(-127, 128, (HIDDEN, (HEADS + 2 * KV) * DIM), generator=g, device=dev, dtype=torch.int8)
        self.o = torch.randint(-127, 128, (HEADS * DIM, HIDDEN), generator=g, device=dev, dtype=torch.int8)
        self.qkv_scale = torch.full((self.qkv.shape[1],), 4e-4, device=dev)
        self.o_scale = torch.full((HIDDEN,), 3e-4, device=dev)
        self.inv_freq = (10000.0 ** (-torch.arange(0, DIM, 2, device=dev, dtype=torch.float64) / DIM)).float()
        self.k, self.v = torch.full((2, pages, PAGE, KV, DIM), 77, dtype=torch.int8, device=dev)
        self.ks, self.vs = torch.full((2, pages, KV, PAGE), float("nan"), device=dev)

    def cache(self):
        return self.k, self.v, self.ks, self.vs

    def __call__(self, x, positions, slots, table, lens, starts=None, **window):
        n = self.npu
        xq, scale, _ = n.npu_rms_norm_dynamic_quant(x, self.gamma)
        qkv = n.npu_quant_matmul(xq, self.qkv, self.qkv_scale, pertoken_scale=scale, output_dtype=self.dtype)
        q, k, v = (t.view(len(x), -1, DIM) for t in qkv.split([HEADS * DIM, KV * DIM, KV * DIM], 1))
        q = n.npu_rotary_axes_quant_cache(q, k, v, positions, self.inv_freq, *self.cache(), slots, sections=[24, 20, 20])
        if starts is None:
            a, lse = n.npu_paged_quant_attention(q, *self.cache(), table, lens, **window)
        else:
            wide = -(-table.shape[1] * PAGE // ROWS)
            rows = torch.arange(len(lens) * wide, dtype=torch.int32, device=self.dev).view(len(lens), wide)
            k_rows, v_rows = torch.full((2, rows.numel(), ROWS, KV, DIM), float("nan"), dtype=self.dtype, device=self.dev)
            n.npu_paged_cache_dequant(*self.cache(), table, lens, k_rows, v_rows, rows)
            a, lse = n.npu_paged_prompt_attention(q, k_rows, v_rows, rows, lens, starts, **window)
        aq, scale = n.npu_dynamic_quant(a.reshape(-1, HEADS * DIM))
        return n.npu_quant_matmul(aq, self.o, self.o_scale, pertoken_scale=scale, output_dtype=self.dtype), a, lse, q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [{}, {"window": 100, "sinks": 4}])
def test_chunks_and_single_tokens(npu, dev, dtype, window):
    lens = [333, 70]
    total, first, singles = sum(lens), [200, 65], 5
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((total, HIDDEN), generator=g, device=dev).to(dtype)
    positions = torch.randint(0, 50000, (3, total), generator=g, device=dev)
    need = [-(-n // PAGE) for n in lens]
    ids = torch.randperm(sum(need) + 5, generator=g, device=dev).int()
    table = torch.full((2, max(need)), -1, dtype=torch.int32, device=dev)
    table[0, :need[0]], table[1, :need[1]] = ids[:need[0]], ids[need[0]:sum(need)]
    place = torch.cat([torch.arange(n, device=dev) for n in lens])
    seq = torch.cat([torch.full((n,), b, device=dev) for b, n in enumerate(lens)])
    slots = table[seq, place // PAGE].long() * PAGE + place % PAGE
    rows = [[i for i in range(total) if seq[i] == b] for b in range(2)]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    layer = Layer(npu, dev, dtype, len(ids))
    whole = layer(x, positions, slots, table, ints(lens), ints([0, lens[0], total]), **window)
    assert bool(whole[0].isfinite().all())
    kept = [t.clone() for t in layer.cache()]

    layer = Layer(npu, dev, dtype, len(ids))
    out = [torch.empty_like(t) for t in whole]

    def step(pick, length, starts):
        at = torch.tensor([i for p in pick for i in p], device=dev)
        for o, t in zip(out, layer(x[at], positions[:, at], slots[at], table, ints(length), starts, **window)):
            o[at] = t

    step([rows[b][:first[b]] for b in range(2)], first, ints([0, first[0], sum(first)]))
    second = [lens[b] - singles for b in range(2)]
    step([rows[b][first[b]:second[b]] for b in range(2)], second, ints([0, second[0] - first[0], sum(second) - sum(first)]))
    for i in range(singles):
        step([[rows[b][second[b] + i]] for b in range(2)], [n + i + 1 for n in second], None)

    # a row's quantization and projection do not depend on the other rows: queries and caches are the same bits
    assert torch.equal(out[3], whole[3])
    assert torch.equal(layer.k, kept[0]) and torch.equal(layer.v, kept[1])
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(layer.cache()[2:], kept[2:]))
    # Prompts: attention over what codes and scales stand for, rounded to the type once more (half a step u of each key and value): scores are off by u of their
    # terms' absolute sum, so weights by 2 u of that and outputs by that and u of sum p |v|, beside the bounds of the attention itself.
    k, v = (oracle.values(layer.k, layer.ks), oracle.values(layer.v, layer.vs))
    ref, ref_lse, weight, spread, reach = paged_oracle.attention(whole[3], k.nan_to_num(), v.nan_to_num(), table, ints(lens), ints([0, lens[0], total]), **window)
    bound, lse_bound = paged_oracle.attention_bounds(dtype, DIM, ref, ref_lse, weight, spread, reach)
    u = torch.finfo(dtype).eps / 2
    bound, lse_bound = bound + (2 * u * reach[..., None] * (1 + 2 * u * reach[..., None]) + u) * weight * (1 + u), lse_bound + u * reach
    for run in (out, whole):
        assert bool(((run[1].double() - ref).abs() <= bound).all())
        assert bool(((run[2].double() - ref_lse).abs() <= lse_bound).all())
    # single tokens, over the cache itself: their own, narrower bounds
    for i in range(singles):
        at = [rows[b][second[b] + i] for b in range(2)]
        one, one_lse, near, lse_near = oracle.attention(out[3][at], *layer.cache(), table, ints([n + i + 1 for n in second]), **window)
        assert bool(((out[1][at].double() - one).abs() <= near).all()) and bool(((out[2][at].double() - one_lse).abs() <= lse_near).all())
