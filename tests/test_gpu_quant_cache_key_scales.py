"""Attention over an int8 cache whose keys are very large or very small, by queries that make up for it: the limits that the header states."""
import math

import pytest
import torch

from test_gpu_quant_cache_attention import LENS, check, make, npu  # noqa: F401  (npu: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("log_size", [90, 86, 40, -40, -100, -120])
def test_sizes_of_keys(npu, dev, dim, log_size):  # noqa: F811
    q, k, v, ks, vs, table, lens = make(dev, LENS, dim=dim, seed=40, size=2.0 ** (-log_size - 6), key_size=2.0 ** (log_size - 3))
    ks = ks.clamp(max=2.0 ** log_size)  # (NaN stays)
    check(npu, q, k, v, ks, vs, table, lens)


def test_scores_of_minus_infinity(npu, dev):
    """A key whose scale is infinite has the score -inf where its sum is negative, and no weight beside finite scores; a row of no other score sees nothing."""
    q, k, v, ks, vs, table, lens = make(dev, [40, 1], heads=1, kv=1, dim=64, seed=41, spare=0)
    q[:], k[:] = 1.0, 1
    clean = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens, window=37, sinks=2)
    k[table[0, 0], 2], ks[table[0, 0], 0, 2] = -1, math.inf  # place 2 of 40, behind the sinks and in front of the window
    got = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens, window=37, sinks=2)
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    k[table[1, 0], 0], ks[table[1, 0], 0, 0] = -1, math.inf
    out, lse = npu.npu_paged_quant_attention(q, k, v, ks, vs, table, lens)
    keep = torch.arange(40, device=dev) != 2
    pages = table[0].long()[torch.arange(40, device=dev) // 16]
    at = torch.arange(40, device=dev) % 16
    x = 64.0 * ks[pages, 0, at].double() * 64 ** -0.5
    p = torch.softmax(x[keep], 0)
    want = (p * vs[pages, 0, at].double()[keep]) @ v[pages, at, 0].double()[keep]
    assert ((out[0, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * (p * vs[pages, 0, at].double()[keep]) @ v[pages, at, 0].double()[keep].abs()).all()
    assert abs(lse[0, 0].item() - torch.logsumexp(x[keep], 0).item()) <= 2.0 ** -16
    assert not out[1].any() and lse[1].item() == -math.inf
