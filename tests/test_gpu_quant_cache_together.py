"""Calls over int8 caches at the same time, and batches of every size that the joining of parts goes by."""
import random

import pytest
import torch

from test_gpu_quant_cache_attention import check, make, npu  # noqa: F401  (npu: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("batch,heads,kv", [(1, 1, 1), (1, 32, 2), (7, 8, 4), (40, 8, 8), (90, 16, 1), (150, 8, 8), (300, 1, 1), (700, 1, 1), (700, 4, 1), (650, 9, 3)])
def test_batches(npu, dev, batch, heads, kv, dim):  # noqa: F811
    """Few and many rows, of items fewer and more than CTAs."""
    rng = random.Random(batch + heads)
    lens = [rng.choice([0, 1, rng.randrange(40), rng.randrange(400)]) for _ in range(batch - 1)] + [777]
    check(npu, *make(dev, lens, heads=heads, kv=kv, dim=dim, page=rng.choice([5, 8, 16, 64]), seed=batch))


def test_two_graphs_at_once(npu, dev):  # noqa: F811
    """Two captured passes (written, attended, read back), replayed on two streams at the same time, over caches of their own."""
    runs = []
    for seed in (31, 32):
        q, k, v, ks, vs, table, lens = make(dev, [300, 2, 0, 1500, 64], heads=16, kv=4, dim=128, seed=seed)
        g = torch.Generator(device=dev).manual_seed(seed)
        new_k, new_v = (torch.randn((5, 4, 128), generator=g, device=dev).to(q.dtype) for _ in range(2))
        positions, inv_freq = (lens - 1).clamp_min(0).long(), (10000.0 ** (-torch.arange(64, device=dev) / 64)).float()
        page = positions // 16
        slots = torch.where(lens > 0, table.gather(1, page[:, None])[:, 0].long() * 16 + positions % 16, -1)
        outs = [torch.zeros((len(k), 16, 4, 128), dtype=q.dtype, device=dev) for _ in range(2)]

        def step(args=(q, new_k, new_v, positions, inv_freq, k, v, ks, vs, slots), cache=(k, v, ks, vs, table, lens), outs=outs):
            turned = npu.npu_rotary_axes_quant_cache(*args)
            out, lse = npu.npu_paged_quant_attention(turned, *cache)
            npu.npu_paged_cache_dequant(*cache, *outs, cache[4])
            return turned, out, lse, *outs

        want = [x.clone() for x in step()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        runs.append((graph, got, want, torch.cuda.Stream(), step))  # (step has the inputs, which the graph does not keep)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, got, _, stream, _ in runs:
            with torch.cuda.stream(stream):
                for x in got:
                    x.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in runs:
        assert all(torch.equal(x, y) for x, y in zip(got, want))
