"""The operators over a paged cache without a GPU: registry, schemas, refusals of the C ABI, and the oracle against loops."""
import ctypes
import math
import sys
from pathlib import Path

import pytest
import torch

from oracle import paged_oracle

ROOT = Path(__file__).resolve().parent.parent
PKG_DIR = ROOT / "ascend-python_b200"


def test_registry(tmp_path):
    sys.path.insert(0, str(PKG_DIR))
    try:
        from codegen import gen_backend_stubs as gen
    finally:
        sys.path.pop(0)
    config = PKG_DIR / "op_plugin" / "config"
    ops = gen.run([config / "op_plugin_functions.yaml", config / "op_plugin_cache_functions.yaml"], tmp_path)
    assert [o.name for o in ops][-4:] == ["npu_rotary_axes", "npu_rotary_axes_cache", "npu_paged_attention",
                                          "npu_paged_prompt_attention"]
    text = (tmp_path / "OpInterface.h").read_text()
    assert "at::IntArrayRef sections={}" in text and "c10::optional<double> scale_value=c10::nullopt" in text
    assert "const at::Tensor &key_cache, const at::Tensor &value_cache" in text
    assert "Tensor(a!) key_cache" in (tmp_path / "TorchLibrary.cpp").read_text()
    with pytest.raises(ValueError):
        gen.parse_schema("f(Tensor(ab!) x) -> Tensor", "op_api")


def test_schemas_and_shim(pkg):
    ops = pkg.load_ops()
    assert str(ops.npu_paged_attention.default._schema) == (
        "npu::npu_paged_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, *, "
        "float? scale_value=None, int window=0, int sinks=0) -> (Tensor, Tensor)")
    schema = ops.npu_rotary_axes_cache.default._schema
    assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == ["key_cache", "value_cache"]
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    x, c, i = torch.zeros((2, 2, 8)), torch.zeros((1, 4, 2, 8)), torch.zeros(2, dtype=torch.int32)
    calls = [lambda: torch_npu.npu_rotary_axes(x, x, i, torch.ones(4)),
             lambda: torch_npu.npu_rotary_axes_cache(x, x, x, i, torch.ones(4), c, c, i),
             lambda: torch_npu.npu_paged_attention(x, c, c, i[:, None], i, scale_value=0.5, window=3, sinks=1),
             lambda: torch_npu.npu_paged_prompt_attention(x, c, c, i[:, None], i, i)]
    for f in calls:  # CPU tensors: no kernel registered
        with pytest.raises(NotImplementedError):
            f()


def _cache(capi, **kw):
    fields = dict(key=1 << 20, value=1 << 21, pages=4, page_size=16, kv_heads=2, dim=64, key_stride_page=2048, key_stride_place=128,
                  key_stride_head=64, value_stride_page=2048, value_stride_place=128, value_stride_head=64)
    return capi.KvCache(**{**fields, **kw})


def _attention(capi, dtype=0, tokens=2, heads=4, st=256, sh=64, cache=None, columns=4, batch=2, scale=1.0, window=0, sinks=0,
               query=1 << 16):
    """Status and message of both entries; the arguments never reach a launch."""
    lib, cache = capi.lib(), cache or _cache(capi)
    a = lib.qmm_paged_attention(query, dtype, tokens, heads, st, sh, cache, None, columns, columns, None, scale, window, sinks, None,
                                None, None, 0, None), lib.qmm_last_error().decode()
    b = lib.qmm_paged_prompt_attention(query, dtype, tokens, heads, st, sh, cache, None, columns, columns, None, None, batch, scale,
                                       window, sinks, None, None, None, 0, None), lib.qmm_last_error().decode()
    return a, b


@pytest.mark.parametrize("what,text", [
    (dict(dtype=2), "bf16 or f16"), (dict(tokens=-1), "non-negative"), (dict(heads=-4), "non-negative"),
    (dict(columns=-1), "non-negative"), (dict(window=-1), "non-negative"), (dict(window=4, sinks=-1), "non-negative"),
    (dict(sinks=2), "with a window only"), (dict(heads=5), "multiple of the cache's"), (dict(scale=math.inf), "finite"),
    (dict(scale=math.nan), "finite"), (dict(query=(1 << 16) + 2), "16-byte"), (dict(st=260), "16-byte"), (dict(sh=4), "16-byte"),
    (dict(heads=70000), "out of range"), (dict(tokens=2**31), "out of range"), (dict(columns=2**31), "out of range")])
def test_attention_refusals(capi, what, text):
    for rc, message in _attention(capi, **what):
        assert rc == 1 and text in message, message


@pytest.mark.parametrize("what,text", [
    (dict(dim=4), "multiple of 8"), (dict(dim=60), "multiple of 8"), (dict(dim=264), "up to 256"), (dict(dim=0), "multiple of 8"),
    (dict(page_size=0), "page size"), (dict(page_size=2**31), "page size"), (dict(pages=-1), "non-negative"),
    (dict(kv_heads=0), "multiple of the cache's"), (dict(pages=2**31), "out of range"), (dict(key=8), "16-byte"),
    (dict(value=1 << 20 | 8), "16-byte"), (dict(key_stride_page=2044), "16-byte"), (dict(value_stride_place=4), "16-byte"),
    (dict(value_stride_head=9), "16-byte")])
def test_cache_refusals(capi, what, text):
    for rc, message in _attention(capi, cache=_cache(capi, **what)):
        assert rc == 1 and text in message, message


def test_empty_calls_launch_nothing(capi):
    lib = capi.lib()
    assert all(rc == 0 for rc, _ in _attention(capi, tokens=0, batch=0))
    assert all(rc == 0 for rc, _ in _attention(capi, heads=0))
    one = (ctypes.c_int64 * 1)(4)
    assert lib.qmm_rotary_axes(None, 0, 0, None, 0, 0, 0, 0, 4, 2, 8, None, 3, 0, 1, None, 4, one, 1, 0, 0, None, None, None) == 0


@pytest.mark.parametrize("what,text", [
    (dict(dtype=3), "bf16, f16 or f32"), (dict(tokens=-1), "non-negative"), (dict(dim=257), "above 256"), (dict(pairs=5), "more frequencies"),
    (dict(pairs=-1), "more frequencies"), (dict(sections=[]), "1 and 8 axes"), (dict(sections=[0] * 9), "1 and 8 axes"),
    (dict(sections=[3]), "add up"), (dict(sections=[2, 3]), "add up"), (dict(sections=[5, -1]), "between 0 and"),
    (dict(sections=[2**62, 2**62]), "between 0 and"), (dict(sections=[0, 4], cyclic=1), "cyclic"), (dict(sections=[1, 2, 1], cyclic=1), "cyclic"),
    (dict(position_dtype=2), "int32 or int64"), (dict(tokens=2**31), "out of range"), (dict(heads=70000), "out of range")])
def test_rotary_refusals(capi, what, text):
    a = {**dict(dtype=0, tokens=2, heads=4, dim=8, pairs=4, sections=[4], cyclic=0, position_dtype=3), **what}
    sections = (ctypes.c_int64 * max(1, len(a["sections"])))(*a["sections"])
    rc = capi.lib().qmm_rotary_axes(None, 32, 8, None, 16, 8, a["dtype"], a["tokens"], a["heads"], 2, a["dim"], None, a["position_dtype"], 2,
                                    1, None, a["pairs"], sections, len(a["sections"]), 0, a["cyclic"], None, None, None)
    assert rc == 1 and text in capi.lib().qmm_last_error().decode()


def test_oracle_against_loops():
    """The oracle's gathered sums against the definition, element by element."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((4, 4, 8), (5, 3, 2, 8), (5, 3, 2, 8)))
    table = torch.tensor([[2, 0, 9], [4, -1, 1]], dtype=torch.int32)
    lens, start = torch.tensor([5, 9], dtype=torch.int32), torch.tensor([0, 1, 3], dtype=torch.int32)
    out, lse, *_ = paged_oracle.attention(q, k, v, table, lens, start, scale=0.5, window=3, sinks=1)
    for t, (b, place) in enumerate([(0, 4), (1, 7), (1, 8), (None, None)]):
        for h in range(4):
            sums, total = [0.0] * 8, 0.0
            for j in range(9):
                if b is None or j > place or not (place - j < 3 or j < 1) or not 0 <= table[b, j // 3] < 5:
                    continue
                e = math.exp(0.5 * float(q[t, h] @ k[table[b, j // 3], j % 3, h // 2]))
                total += e
                sums = [s + e * float(x) for s, x in zip(sums, v[table[b, j // 3], j % 3, h // 2])]
            if total == 0:
                assert lse[t, h] == -math.inf and not out[t, h].any()
            else:
                assert abs(float(lse[t, h]) - math.log(total)) < 1e-12
                assert all(abs(float(x) - s / total) < 1e-12 for x, s in zip(out[t, h], sums))
    x = torch.randn((3, 2, 10), generator=g, dtype=torch.float64)
    positions, freq = torch.tensor([[1, 2, 3], [4, 5, 60]]), torch.tensor([1.0, 0.5, 0.25, 0.125])
    for cyclic, axes in ((False, [0, 0, 0, 1]), (True, [0, 1, 0, 0])):
        for interleaved in (False, True):
            y = paged_oracle.rotary(x, positions, freq, [3, 1], interleaved, cyclic)
            for t in range(3):
                for i, a in enumerate(axes):
                    m, n = (2 * i, 2 * i + 1) if interleaved else (i, i + 4)
                    angle = float(positions[a, t]) * float(freq[i])
                    z = complex(x[t, 1, m], x[t, 1, n]) * complex(math.cos(angle), math.sin(angle))
                    assert abs(float(y[t, 1, m]) - z.real) < 1e-12 and abs(float(y[t, 1, n]) - z.imag) < 1e-12
            assert torch.equal(y[..., 8:], x[..., 8:])


def test_short_cut_calls_are_the_operators(pkg):
    """What the shim's positional calls leave to torch.ops, and that what they take reaches the operator."""
    from torch.utils._python_dispatch import TorchDispatchMode

    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func.namespace != "npu":
                return func(*args, **(kwargs or {}))
            seen.append((func.name().split("::")[1], len(args) + len(kwargs or {})))
            return tuple(torch.zeros(1) for _ in func._schema.returns) if len(func._schema.returns) > 1 else torch.zeros(1)

    x, c, i, f = torch.zeros((2, 2, 8)), torch.zeros((1, 4, 2, 8)), torch.zeros(2, dtype=torch.int32), torch.ones(4)
    calls = {"npu_rotary_axes": [lambda **k: torch_npu.npu_rotary_axes(x, x, i, f, **k), {}, {"sections": [4]}, {"sections": (4,)},
                                 {"rotary_mode": "interleave", "axis_order": "cyclic"}],
             "npu_rotary_axes_cache": [lambda **k: torch_npu.npu_rotary_axes_cache(x, x, x, i, f, c, c, i, **k), {}, {"sections": [4]}],
             "npu_paged_attention": [lambda **k: torch_npu.npu_paged_attention(x, c, c, i[:, None], i, **k), {}, {"scale_value": 0.5},
                                     {"scale_value": 1, "window": 3, "sinks": 2}],
             "npu_paged_prompt_attention": [lambda **k: torch_npu.npu_paged_prompt_attention(x, c, c, i[:, None], i, i, **k), {}, {"window": 3}]}
    for name, (call, *options) in calls.items():
        for option in options:
            seen = []
            with Record():
                call(**option)
            assert [n for n, _ in seen] == [name]
    for bad in ({"sections": [1.5]}, {"sections": 4.0}, {"rotary_mode": 3}):
        with pytest.raises((RuntimeError, TypeError)):
            torch_npu.npu_rotary_axes(x, x, i, f, **bad)
    with pytest.raises((RuntimeError, TypeError)):
        torch_npu.npu_paged_attention(x, c, c, i[:, None], i, window="x")


def test_workspace_sizes(capi):
    """The scratch is bounded by the GPU, not by the batch or the cache, where sums of tokens are not kept; and grows with what is."""
    lib, n = capi.lib(), ctypes.c_size_t(0)

    def decode(*a):
        assert lib.qmm_paged_attention_workspace_size(*a, ctypes.byref(n)) == 0
        return n.value

    def prompt(*a):
        assert lib.qmm_paged_prompt_attention_workspace_size(*a, ctypes.byref(n)) == 0
        return n.value

    assert decode(0, 8, 2, 64, 100) == 0 and decode(4, 0, 2, 64, 100) == 0
    assert decode(1, 64, 8, 128, 1 << 20) == decode(4096, 64, 8, 128, 1 << 20) <= 40 << 20
    assert prompt(0, 0, 8, 2, 64, 100) == 0
    assert prompt(100000, 10, 32, 8, 128, 1 << 17) == 0          # enough tiles for every SM: nothing is split
    assert prompt(4, 1, 32, 8, 128, 400) == 0                     # short: nothing to split
    assert 0 < prompt(2000, 1, 32, 8, 128, 1 << 20) <= (256 << 20) * 130 // 128
    few = prompt(4, 1, 32, 8, 128, 1 << 17)
    assert 0 < few <= 64 * 4 * 32 * (128 + 2) * 4 + 16
    assert lib.qmm_paged_attention_workspace_size(-1, 8, 2, 64, 100, ctypes.byref(n)) == 1
    assert lib.qmm_paged_prompt_attention_workspace_size(4, 1, 8, 0, 64, 100, ctypes.byref(n)) == 1


@pytest.mark.gpu
def test_workspaces_that_are_too_small(capi, dev):
    """A scratch that is missing, too small or off its alignment is refused before any launch."""
    lib = capi.lib()
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16, device=dev)
    q, out, lse = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev), torch.empty((2, 4, 64), dtype=torch.bfloat16, device=dev), torch.empty((2, 4), device=dev)
    table, lens, start = torch.zeros((2, 100), dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev), torch.arange(3, dtype=torch.int32, device=dev)
    n = ctypes.c_size_t(0)
    lib.qmm_paged_attention_workspace_size(2, 4, 2, 64, 1600, ctypes.byref(n))
    scratch = torch.empty(n.value + 16, dtype=torch.uint8, device=dev)
    for pointer, size in ((None, n.value), (scratch.data_ptr(), n.value - 1), (scratch.data_ptr() + 8, n.value)):
        rc = lib.qmm_paged_attention(q.data_ptr(), 0, 2, 4, 256, 64, capi.kv_cache(cache, cache), table.data_ptr(), 100, 100, lens.data_ptr(), 1.0,
                                     0, 0, out.data_ptr(), lse.data_ptr(), pointer, size, None)
        assert rc == 6 and b"workspace" in lib.qmm_last_error()
    lib.qmm_paged_prompt_attention_workspace_size(2, 2, 4, 2, 64, 1600, ctypes.byref(n))
    assert n.value > 0
    rc = lib.qmm_paged_prompt_attention(q.data_ptr(), 0, 2, 4, 256, 64, capi.kv_cache(cache, cache), table.data_ptr(), 100, 100, lens.data_ptr(),
                                        start.data_ptr(), 2, 1.0, 0, 0, out.data_ptr(), lse.data_ptr(), scratch.data_ptr(), n.value - 1, None)
    assert rc == 6 and b"workspace" in lib.qmm_last_error()
