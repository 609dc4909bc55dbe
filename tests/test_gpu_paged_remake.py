"""Prompts whose rows come beside values that are not finite and that they do not see: such rows are made again when a CTA's items are
done, and neither they nor the items behind them, of other sequences and heads, are touched by those values."""
import ctypes
import math
import random

import pytest
import torch

from test_gpu_paged_attention import call, make, npu, paged  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def compare(paged, out, lse, q, k, v, table, lens, starts, only, **kw):
    """Rows `only` against the definition: NaN and infinities where it has them, the rest within its bounds."""
    ref = paged.attention(q, k, v, table, lens, starts, only=only, **kw)
    bound, lse_bound = paged.attention_bounds(q.dtype, q.shape[2], *ref)
    rows = torch.tensor(sorted(only), device=q.device)
    want, got, bound = ref[0][rows], out.double()[rows], bound[rows]
    odd = ~want.isfinite()
    assert torch.equal(got[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), want[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
    assert bool(((got - want).abs() <= bound)[~odd].all())
    none = ref[1][rows] == -math.inf
    assert torch.equal((lse == -math.inf)[rows], none)
    assert bool(((lse.double() - ref[1]).abs() <= lse_bound)[rows][~none].all())
    return int(odd.sum())


def nothing_is_split(capi, q, k, table, lens):
    n = ctypes.c_size_t(0)
    assert capi.lib().qmm_paged_prompt_attention_workspace_size(q.shape[0], lens.numel(), q.shape[1], k.shape[2], q.shape[2],
                                                                table.shape[1] * k.shape[1], ctypes.byref(n)) == 0
    return n.value == 0


@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float16), (256, torch.bfloat16)])
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_a_value_late_in_a_long_sequence(npu, paged, capi, dev, poison, dim, dtype):
    """4000 places, in a batch that leaves nothing to split: finite sequences come behind it."""
    new = [900] + [100] * 40
    lens = [4000] + [200] * 40
    q, k, v, table, length, starts = make(dev, lens, new, heads=16, kv=8, dim=dim, dtype=dtype, seed=31)
    assert nothing_is_split(capi, q, k, table, length)
    clean = call(npu, q, k, v, table, length, starts)
    for j in (3500, 3973):
        v2 = v.clone()
        v2[table[0, j // 16], j % 16, 1::3, 5] = poison
        out, lse = call(npu, q, k, v2, table, length, starts)
        assert torch.equal(lse, clean[1]) and torch.equal(out[900:], clean[0][900:])
        near = j - 3100
        only = set(random.Random(j).sample(range(900), 40)) | set(range(max(0, near - 130), min(900, near + 20), 3))
        assert compare(paged, out, lse, q, k, v2, table, length, starts, only) > 0


@pytest.mark.parametrize("heads,kv,dim,page,dtype", [(16, 8, 128, 16, torch.bfloat16), (8, 8, 64, 8, torch.float16), (16, 4, 256, 32, torch.bfloat16),
                                                     (28, 4, 128, 20, torch.float16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_such_values_in_every_sequence(npu, paged, capi, dev, window, sinks, heads, kv, dim, page, dtype):
    """Every CTA meets them in its first items, and the blocks that it does not go on to are as many again."""
    rng = random.Random(dim)
    new = [rng.choice([1, 7, 60, 130, 200]) for _ in range(150)]
    lens = [n + rng.randrange(150) for n in new]
    q, k, v, table, length, starts = make(dev, lens, new, heads=heads, kv=kv, dim=dim, page=page, dtype=dtype, seed=dim + page, tail=5)
    assert nothing_is_split(capi, q, k, table, length)
    for b, n in enumerate(lens):
        j = n - 1 - new[b] // 2
        v[table[b, j // page], j % page, :, 3] = (math.nan, math.inf, -math.inf)[b % 3]
    out, lse = call(npu, q, k, v, table, length, starts, window=window, sinks=sinks)
    only = set(rng.sample(range(q.shape[0]), 400)) | {0, q.shape[0] - 1}
    assert compare(paged, out, lse, q, k, v, table, length, starts, only, window=window, sinks=sinks) > 0
    again = call(npu, q, k, v, table, length, starts, window=window, sinks=sinks)
    assert torch.equal(out.nan_to_num(nan=7.0), again[0].nan_to_num(nan=7.0)) and torch.equal(lse, again[1])


def test_in_a_graph(npu, dev):
    """A captured call whose values are, are not, and are again finite."""
    q, k, v, table, length, starts = make(dev, [400] * 60, [130] * 60, heads=8, kv=8, dim=128, seed=33)
    state = (q, k, v, table, length, starts)
    call(npu, *state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(npu, *state)
    finite = v.clone()
    for poison in (None, math.nan, None, math.inf):
        v.copy_(finite)
        if poison is not None:
            v[table[:, 20], 3, :, 7] = poison
        graph.replay()
        want = call(npu, *state)
        assert torch.equal(got[0].nan_to_num(nan=7.0), want[0].nan_to_num(nan=7.0)) and torch.equal(got[1], want[1])
        assert bool(got[0].isfinite().all()) == (poison is None)
