"""Attention with scores of 2^21, the largest that its operators are for, equal ones for all keys: they share the weight."""
import math
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"
PAGE, LENS = 16, [1, 16, 40, 300]


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


@pytest.mark.parametrize("kind", ["single", "prompt", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("score", [2.0 ** 21, -2.0 ** 21, 1.7e6, -1.3e6, 98765.4])
def test_equal_scores(npu, dev, score, dim, dtype, kind):
    """A score is scale_value times 256, times log2(e) in fp32, off by 2^-23 of it at most, as is the log-sum.  Weights are rounded to the type of the
    values (bf16 where a 16-bit cache is), half a step each way, and the output once."""
    g = torch.Generator(device=dev).manual_seed(dim)
    pages = sum(-(-n // PAGE) for n in LENS)
    table, at = torch.full((len(LENS), 19), -1, dtype=torch.int32), 0
    for b, n in enumerate(LENS):
        need = -(-n // PAGE)
        table[b, :need] = torch.arange(at, at + need)
        at += need
    lens = torch.tensor(LENS, dtype=torch.int32, device=dev)
    codes = torch.randint(1, 128, (pages, PAGE, 1, dim), generator=g, device=dev, dtype=torch.int8)
    k = torch.zeros_like(codes)
    k[..., 0] = 16
    q = torch.zeros((len(LENS), 4, dim), dtype=dtype, device=dev)
    q[..., 0] = 16.0
    scale = score / 256.0
    if kind == "int8":
        ones = torch.ones((pages, 1, PAGE), device=dev)
        out, lse = npu.npu_paged_quant_attention(q, k, codes, ones, ones, table.to(dev), lens, scale_value=scale)
    elif kind == "single":
        out, lse = npu.npu_paged_attention(q, k.to(dtype), codes.to(dtype), table.to(dev), lens, scale_value=scale)
    else:
        start = torch.arange(len(LENS) + 1, dtype=torch.int32, device=dev)
        out, lse = npu.npu_paged_prompt_attention(q, k.to(dtype), codes.to(dtype), table.to(dev), lens, start, scale_value=scale)
    for b, n in enumerate(LENS):
        values = codes[table[b].long()].flatten(0, 1)[:n, 0].double()
        err = (out[b].double() / values.mean(0) - 1).abs().max().item()
        assert err <= 3 * torch.finfo(dtype).eps / 2 + 2.0 ** -11, (n, err)
        assert (lse[b].double() / (score + math.log(n)) - 1).abs().max().item() <= 2.0 ** -22
