"""Attention over an int8 cache where a warp has hundreds of thousands of places of a sequence: sums that stay exact over long stretches."""
import math
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"
PAGE, DISTINCT, BATCH = 4096, 16, 301


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


def make(dev, places, heads, kv, dim, dtype, rise, seed=0):
    """Sequences that name the same pages again and again, the last page's keys with scores that are higher by `rise`."""
    g = torch.Generator(device=dev).manual_seed(seed)
    k = torch.randint(-60, 61, (DISTINCT + 1, PAGE, kv, dim), generator=g, device=dev, dtype=torch.int8)
    v = torch.randint(30, 128, (DISTINCT + 1, PAGE, kv, dim), generator=g, device=dev, dtype=torch.int8)
    ks = torch.full((DISTINCT + 1, kv, PAGE), 0.01, device=dev)
    vs = 0.01 + 0.01 * torch.rand((DISTINCT + 1, kv, PAGE), generator=g, device=dev)
    q = torch.randn((BATCH, heads, dim), generator=g, device=dev).to(dtype)
    q[..., 0] = 1.0
    k[..., 0] = 0
    k[DISTINCT, :, :, 0] = round(min(127.0, rise * math.sqrt(dim) / 0.01))
    table = (torch.arange(places // PAGE, device=dev) % DISTINCT).int().repeat(BATCH, 1)
    table[:, -1] = DISTINCT
    return q, k, v, ks, vs, table, torch.full((BATCH,), places, dtype=torch.int32, device=dev)


def definition(q, k, v, ks, vs, table, row):
    times = torch.bincount(table[0].long(), minlength=len(k)).double().repeat_interleave(PAGE)
    group = q.shape[1] // k.shape[2]
    keys, values = ((x.double() * s.double().transpose(1, 2)[..., None]).flatten(0, 1).repeat_interleave(group, 1) for x, s in ((k, ks), (v, vs)))
    x = torch.einsum("hd,nhd->hn", q[row].double(), keys) * q.shape[2] ** -0.5
    lse = torch.logsumexp(x + times.log(), 1)
    p = torch.exp(x - lse[:, None]) * times
    return torch.einsum("hn,nhd->hd", p, values), lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim,log_places", [(4, 1, 64, 21), (20, 1, 128, 21), (2, 1, 256, 21), (3, 1, 80, 20), (8, 4, 64, 18), (6, 2, 128, 20), (9, 1, 256, 20)])
@pytest.mark.parametrize("rise", [0.0, 0.1])
def test_long_sums(npu, dev, heads, kv, dim, log_places, rise, dtype):
    """A weight is rounded to f16 (2^-11, by chance alike), the output to its type (half a step u); sums over stretches of 2^16 to 2^17 places lose up to
    2^-11, all towards 0, and scores' roundings are 2^-24 of some 16 at most."""
    args = make(dev, 1 << log_places, heads, kv, dim, dtype, rise, seed=dim + heads)
    args[6][5:9] = torch.tensor([1, 3, 0, 1], device=dev)
    out, lse = npu.npu_paged_quant_attention(*args)
    u = torch.finfo(dtype).eps / 2
    for row in (0, 1, 4, 9, 77, 150, 300):
        want, want_lse = definition(*args[:6], row)
        assert ((out[row].double() / want - 1).abs().max().item()) <= u + 2.0 ** -10 + 2.0 ** -12
        assert (lse[row].double() - want_lse).abs().max().item() <= 2.0 ** -12
    assert not out[7].any() and bool((lse[7] == -math.inf).all()) and bool(out.isfinite().all())
