"""A prompt's item that takes longer than the limit of the waits inside a CTA."""
import math

import pytest
import torch

from test_gpu_paged_attention import npu  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def test_two_to_the_29_places_in_one_item(npu, capi, dev):
    """A table that names one page 8192 times, beside enough short sequences that nothing is split: one CTA works for some seconds.
    Keys of 0 and values of powers of two make every sum exact."""
    page, columns, batch = 65536, 8192, 301
    k = torch.zeros((1, page, 1, 8), dtype=torch.bfloat16, device=dev)
    v = (2.0 ** torch.arange(-3, 5, device=dev)).to(torch.bfloat16).expand(1, page, 1, 8).contiguous()
    table = torch.zeros((batch, columns), dtype=torch.int32, device=dev)
    lens = torch.ones(batch, dtype=torch.int32, device=dev)
    lens[0] = page * columns
    starts = torch.arange(batch + 1, dtype=torch.int32, device=dev)
    out, lse = npu.npu_paged_prompt_attention(torch.ones((batch, 1, 8), dtype=torch.bfloat16, device=dev), k, v, table, lens, starts)
    torch.cuda.synchronize()
    assert capi.device_status() == 0
    assert torch.equal(out, v[0, :1].expand(batch, 1, 8))
    assert abs(lse[0].item() - math.log(page * columns)) <= 2.0 ** -18 and bool((lse[1:] == 0).all())
