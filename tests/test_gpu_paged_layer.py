"""The operators of a quantized decoder layer in a row, as a server runs them: normalisation and quantization, the fused QKV
projection, rotary positions with the cache write, attention over the cache, quantization, the output projection; a prompt in two
chunks, then single tokens, against the prompt in one piece."""
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"
HEADS, KV, DIM, HIDDEN, PAGE = 16, 4, 128, 1024, 16


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
        self.npu, self.dtype = npu, dtype
        self.gamma = (1 + 0.1 * torch.randn(HIDDEN, generator=g, device=dev)).to(dtype)
        self.qkv = torch.randint(-127, 128, (HIDDEN, (HEADS + 2 * KV) * DIM), generator=g, device=dev, dtype=torch.int8)
        self.o = torch.randint(-127, 128, (HEADS * DIM, HIDDEN), generator=g, device=dev, dtype=torch.int8)
        self.qkv_scale = torch.full((self.qkv.shape[1],), 4e-4, device=dev)
        self.o_scale = torch.full((HIDDEN,), 3e-4, device=dev)
        self.inv_freq = (10000.0 ** (-torch.arange(0, DIM, 2, device=dev, dtype=torch.float64) / DIM)).float()
        self.k, self.v = torch.full((2, pages, PAGE, KV, DIM), float("nan"), dtype=dtype, device=dev)

    def __call__(self, x, positions, slots, table, lens, starts=None, **window):
        n = self.npu
        xq, scale, _ = n.npu_rms_norm_dynamic_quant(x, self.gamma)
        qkv = n.npu_quant_matmul(xq, self.qkv, self.qkv_scale, pertoken_scale=scale, output_dtype=self.dtype)
        q, k, v = qkv.split([HEADS * DIM, KV * DIM, KV * DIM], 1)
        q = n.npu_rotary_axes_cache(q.view(-1, HEADS, DIM), k.view(-1, KV, DIM), v.view(-1, KV, DIM), positions, self.inv_freq, self.k,
                                    self.v, slots, sections=[24, 20, 20])
        if starts is None:
            a, lse = n.npu_paged_attention(q, self.k, self.v, table, lens, **window)
        else:
            a, lse = n.npu_paged_prompt_attention(q, self.k, self.v, table, lens, starts, **window)
        aq, scale = n.npu_dynamic_quant(a.reshape(-1, HEADS * DIM))
        return n.npu_quant_matmul(aq, self.o, self.o_scale, pertoken_scale=scale, output_dtype=self.dtype), a, lse, q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [{}, {"window": 100, "sinks": 4}])
def test_chunks_and_single_tokens(npu, dev, dtype, window):
    from oracle import paged_oracle

    lens = [333, 70]
    total, first = sum(lens), [200, 65]
    singles = 5
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

    # a row's quantization and projection do not depend on the other rows, so queries and caches are the same bits
    assert torch.equal(out[3], whole[3])
    ref = paged_oracle.attention(whole[3], layer.k, layer.v, table, ints(lens), ints([0, lens[0], total]), **window)
    bound, lse_bound = paged_oracle.attention_bounds(dtype, DIM, *ref)
    for run in (out, whole):
        assert bool(((run[1].double() - ref[0]).abs() <= bound).all())
        assert bool(((run[2].double() - ref[1]).abs() <= lse_bound).all())
    # the projection of what differs by attention's bounds: at most 2 of them and a quantization step for every input
    a = ref[0].reshape(total, -1)
    step_size = a.abs().amax(1, keepdim=True) * (1 + 2.0 ** -7) / 127
    spread = (2 * bound.reshape(total, -1) + step_size).sum(1, keepdim=True) * 127 * 3e-4
    u = torch.finfo(dtype).eps
    assert bool(((out[0].double() - whole[0].double()).abs() <= spread + u * whole[0].double().abs()).all())
