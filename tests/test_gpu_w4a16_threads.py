"""W4A16 calls from several threads, of sizes that take different amounts of shared memory."""
import sys
import threading
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PKG_DIR = Path(__file__).resolve().parent.parent / "ascend-python_b200"


@pytest.fixture(scope="module")
def npu():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


# rows, K, N of each thread: few rows (weights in any layout), up to 64 and more in the packed one, and one token over long and short runs of blocks
@pytest.mark.parametrize("sizes", [[(20, 1024, 1024), (33, 1024, 1024), (64, 2048, 512), (17, 512, 1024)],
                                   [(100, 1024, 2048), (300, 512, 1024), (150, 2048, 512), (1000, 512, 512)],
                                   [(1, 16384, 16384), (1, 512, 8192), (2, 16384, 16384), (2, 2048, 8192)]])
@pytest.mark.parametrize("group", [128, 32])
def test_threads(npu, dev, sizes, group):
    failed, begin = [], threading.Barrier(len(sizes))

    def work(seed, M, K, N):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                g = torch.Generator(device=dev).manual_seed(seed)
                x = torch.randn((M, K), generator=g, device=dev).to(torch.bfloat16)
                weight = torch.randint(-2**31, 2**31 - 1, (K, N // 8), generator=g, device=dev, dtype=torch.int64).int()
                scale = (torch.rand((K // group, N), generator=g, device=dev) * 0.01).to(x.dtype)
                call = lambda: npu.npu_weight_quant_batchmatmul(x, weight, scale, None, antiquant_group_size=group)  # noqa: E731
                want = [call() for _ in range(3)][-1]
                begin.wait()
                for _ in range(1000):
                    got = call()
                torch.cuda.current_stream().synchronize()
                assert torch.equal(got, want)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)
            begin.abort()

    threads = [threading.Thread(target=work, args=(n, *size)) for n, size in enumerate(sizes)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
