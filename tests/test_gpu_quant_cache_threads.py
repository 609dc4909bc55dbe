"""Calls over int8 caches from several threads, whose kernels take different amounts of shared memory."""
import threading

import pytest
import torch

from test_gpu_quant_cache_attention import make, npu  # noqa: F401  (npu: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_two_threads(npu, dev, dim):  # noqa: F811
    """8 and 2 key-value heads: a CTA's warps have a head each, or parts of its places, which they add up in shared memory."""
    failed, begin = [], threading.Barrier(4)

    def work(seed, kv):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                args = make(dev, [90, 3, 400], heads=8, kv=kv, dim=dim, seed=seed)
                want = npu.npu_paged_quant_attention(*args)
                begin.wait()
                for _ in range(2000):
                    got = npu.npu_paged_quant_attention(*args)
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(x, y) for x, y in zip(got, want))
        except BaseException as e:  # noqa: BLE001
            failed.append(e)
            begin.abort()

    threads = [threading.Thread(target=work, args=(n, kv)) for n, kv in enumerate((8, 2, 8, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
