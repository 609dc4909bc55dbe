"""The write into a paged cache whose storage another tensor has until one of them is written."""
import pytest
import torch

from test_gpu_paged_attention import npu  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def test_lazy_clones_of_a_cache(npu, dev):
    """Of a cache and its lazy clone the one that is written gets storage of its own: the other keeps what it held."""
    k, v = torch.zeros((2, 3, 4, 2, 64), dtype=torch.bfloat16, device=dev)
    x = torch.ones((2, 2, 64), dtype=torch.bfloat16, device=dev)
    at = torch.tensor([1, 6], device=dev)
    for written in range(2):
        k0, v0 = k.clone(), v.clone()
        pairs = [(k0, v0), (torch._lazy_clone(k0), torch._lazy_clone(v0))]
        npu.npu_rotary_axes_cache(x, x, x, at, torch.ones(32, device=dev), *pairs[written], at)
        for (i, pair) in enumerate(pairs):
            for t in pair:
                assert bool(t.ne(0).any()) == (i == written)
