"""The operators over an int8 paged cache without a GPU: registry, schemas, short-cut calls, refusals of the C ABI, the oracle."""
import ctypes
import math
import sys
from pathlib import Path

import pytest
import torch

from oracle import quant_cache_oracle as oracle

ROOT = Path(__file__).resolve().parent.parent
PKG_DIR = ROOT / "ascend-python_b200"
NAMES = ["npu_rotary_axes_quant_cache", "npu_paged_quant_attention", "npu_paged_cache_dequant"]


def _shim():
    sys.path.insert(0, str(PKG_DIR))
    try:
        import torch_npu
    finally:
        sys.path.pop(0)
    return torch_npu


def test_registry(tmp_path):
    sys.path.insert(0, str(PKG_DIR))
    try:
        from codegen import gen_backend_stubs as gen
    finally:
        sys.path.pop(0)
    ops = gen.run([PKG_DIR / "op_plugin" / "config" / "op_plugin_quant_cache_functions.yaml"], tmp_path)
    assert [o.name for o in ops] == NAMES
    assert "void npu_paged_cache_dequant(" in (tmp_path / "OpInterface.h").read_text()
    assert "Tensor(b!) value_out" in (tmp_path / "TorchLibrary.cpp").read_text()
    assert gen.parse_schema("f(Tensor x) -> ()", "op_api").cpp_return() == "void"


def test_schemas_and_shim(pkg):
    ops = pkg.load_ops()
    assert str(ops.npu_paged_quant_attention.default._schema) == (
        "npu::npu_paged_quant_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor key_scale, Tensor value_scale, "
        "Tensor block_table, Tensor seq_lens, *, float? scale_value=None, int window=0, int sinks=0) -> (Tensor, Tensor)")
    written = {"npu_rotary_axes_quant_cache": ["key_cache", "value_cache", "key_scale", "value_scale"], "npu_paged_cache_dequant": ["key_out", "value_out"]}
    for name, want in written.items():
        schema = getattr(ops, name).default._schema
        assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == want
    npu = _shim()
    for call in _calls(npu).values():  # CPU tensors: no kernel registered
        with pytest.raises(NotImplementedError):
            call()


def _calls(npu):
    x, c, i, f = torch.zeros((2, 2, 16)), torch.zeros((1, 4, 2, 16), dtype=torch.int8), torch.zeros(2, dtype=torch.int32), torch.ones(8)
    s, o = torch.zeros((1, 2, 4)), torch.zeros((1, 4, 2, 16))
    return {"npu_rotary_axes_quant_cache": lambda **k: npu.npu_rotary_axes_quant_cache(x, x, x, i, f, c, c, s, s, i, **k),
            "npu_paged_quant_attention": lambda **k: npu.npu_paged_quant_attention(x, c, c, s, s, i[:, None], i, **k),
            "npu_paged_cache_dequant": lambda **k: npu.npu_paged_cache_dequant(c, c, s, s, i[:, None], i, o, o, i[:, None], **k)}


def test_short_cut_calls_are_the_operators(pkg):
    """What the shim's positional calls leave to torch.ops, and that what they take reaches the operator."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func.namespace != "npu":
                return func(*args, **(kwargs or {}))
            seen.append(func.name().split("::")[1])
            n = len(func._schema.returns)
            return tuple(torch.zeros(1) for _ in range(n)) if n > 1 else torch.zeros(1) if n else None

    options = {"npu_rotary_axes_quant_cache": [{}, {"sections": [8]}, {"sections": (8,), "rotary_mode": "interleave"}],
               "npu_paged_quant_attention": [{}, {"scale_value": 0.5}, {"scale_value": 1, "window": 3, "sinks": 2}],
               "npu_paged_cache_dequant": [{}, {"first_places": torch.zeros(2, dtype=torch.int32)}]}
    npu = _shim()
    for name, call in _calls(npu).items():
        for option in options[name]:
            seen = []
            with Record():
                got = call(**option)
            assert seen == [name] and (got is None) == (name == "npu_paged_cache_dequant")
    for bad in ({"window": "x"}, {"sinks": 1.5}, {"scale_value": "x"}):
        with pytest.raises((RuntimeError, TypeError)):
            _calls(npu)["npu_paged_quant_attention"](**bad)


def _cache(capi, **kw):
    fields = dict(key=1 << 20, value=1 << 21, pages=4, page_size=16, kv_heads=2, dim=64, key_stride_page=2048, key_stride_place=128,
                  key_stride_head=64, value_stride_page=2048, value_stride_place=128, value_stride_head=64)
    return capi.KvCache(**{**fields, **kw})


def _scales(capi, **kw):
    fields = dict(key=1 << 22, value=1 << 23, key_stride_page=32, key_stride_place=1, key_stride_head=16, value_stride_page=32,
                  value_stride_place=1, value_stride_head=16)
    return capi.KvScales(**{**fields, **kw})


def _attention(capi, dtype=0, batch=2, heads=4, st=256, sh=64, cache=None, scales=None, columns=4, scale=1.0, window=0, sinks=0,
               query=1 << 16, table=None, lens=None, out=None, lse=None):
    """Status and message; the arguments never reach a launch."""
    lib = capi.lib()
    rc = lib.qmm_paged_quant_attention(query, dtype, batch, heads, st, sh, cache or _cache(capi), scales or _scales(capi), table, columns, columns,
                                       lens, scale, window, sinks, out, lse, None, 0, None)
    return rc, lib.qmm_last_error().decode()


@pytest.mark.parametrize("what,text", [
    (dict(dtype=2), "bf16 or f16"), (dict(batch=-1), "non-negative"), (dict(heads=-4), "non-negative"), (dict(columns=-1), "non-negative"),
    (dict(window=-1), "non-negative"), (dict(window=4, sinks=-1), "non-negative"), (dict(sinks=2), "with a window only"),
    (dict(heads=5), "multiple of the cache's"), (dict(scale=math.inf), "finite"), (dict(scale=math.nan), "finite"), (dict(scale=3e38), "finite"),
    (dict(query=(1 << 16) + 2), "16-byte"), (dict(st=260), "16-byte"), (dict(sh=4), "16-byte"), (dict(heads=70000), "out of range"),
    (dict(batch=2**31), "out of range"), (dict(columns=2**31), "out of range"), (dict(out=8), "boundaries"), (dict(lse=2), "boundaries"),
    (dict(table=2), "boundaries"), (dict(lens=1), "boundaries")])
def test_attention_refusals(capi, what, text):
    rc, message = _attention(capi, **what)
    assert rc == 1 and text in message, message


@pytest.mark.parametrize("what,text", [
    (dict(dim=8), "multiple of 16"), (dict(dim=72), "multiple of 16"), (dict(dim=272), "up to 256"), (dict(dim=0), "multiple of 16"),
    (dict(page_size=0), "page size"), (dict(page_size=2**31), "page size"), (dict(pages=-1), "non-negative"),
    (dict(kv_heads=0), "multiple of the cache's"), (dict(pages=2**31), "out of range"), (dict(key=8), "16-byte"),
    (dict(value=1 << 20 | 8), "16-byte"), (dict(key_stride_page=2040), "16-byte"), (dict(value_stride_place=8), "16-byte"),
    (dict(value_stride_head=9), "16-byte")])
def test_attention_cache_refusals(capi, what, text):
    rc, message = _attention(capi, cache=_cache(capi, **what))
    assert rc == 1 and text in message, message


def test_attention_scales_refusals(capi):
    for what in (dict(key=2), dict(value=1 << 23 | 1)):
        rc, message = _attention(capi, scales=_scales(capi, **what))
        assert rc == 1 and "4-byte" in message
    lib = capi.lib()
    rc = lib.qmm_paged_quant_attention(1 << 16, 0, 2, 4, 256, 64, _cache(capi), None, None, 4, 4, None, 1.0, 0, 0, None, None, None, 0, None)
    assert rc == 1 and "no scales" in lib.qmm_last_error().decode()
    assert _attention(capi, batch=0)[0] == 0 and _attention(capi, heads=0)[0] == 0


def _write(capi, dtype=0, tokens=2, pairs=32, sections=(32,), axes=1, position_dtype=3, slot_dtype=3, cache=None, scales=None):
    lib = capi.lib()
    rc = lib.qmm_rotary_axes_quant_cache(None, 0, 0, None, 0, 0, None, 0, 0, dtype, tokens, 4, None, position_dtype, 0, 1, None, pairs,
                                         (ctypes.c_int64 * len(sections))(*sections), axes, 0, 0, cache or _cache(capi), scales or _scales(capi), None,
                                         slot_dtype, 1, None, None)
    return rc, lib.qmm_last_error().decode()


def test_write_refusals(capi):
    for what, text in ((dict(dtype=3), "bf16, f16 or f32"), (dict(tokens=-1), "non-negative"), (dict(pairs=33), "more frequencies"),
                       (dict(sections=(31,)), "add up"), (dict(axes=9, sections=(0,) * 9), "1 and 8 axes"), (dict(position_dtype=2), "int32 or int64"),
                       (dict(slot_dtype=2), "int32 or int64"), (dict(tokens=2**31), "out of range"),
                       (dict(cache=_cache(capi, value=1 << 20)), "same address"), (dict(scales=_scales(capi, value=1 << 22)), "same address"),
                       (dict(scales=_scales(capi, key=2)), "4-byte"), (dict(cache=_cache(capi, page_size=0)), "size positive"),
                       (dict(cache=_cache(capi, pages=-1)), "non-negative"), (dict(cache=_cache(capi, dim=257)), "above 256")):
        rc, message = _write(capi, **what)
        assert rc == 1 and text in message, (what, message)
    assert _write(capi, tokens=0)[0] == 0
    assert _write(capi, tokens=0, cache=_cache(capi, pages=0, key=None, value=None), scales=_scales(capi, key=None, value=None))[0] == 0


def _read(capi, batch=2, pages=4, out_pages=4, cache=None, scales=None, out=None, out_dtype=0, table=None, out_table=None, lens=None, first=None):
    lib = capi.lib()
    rc = lib.qmm_paged_cache_dequant(cache or _cache(capi), scales or _scales(capi), table, 4, pages, lens, first, batch,
                                     out or _cache(capi, key=1 << 24, value=1 << 25), out_dtype, out_table, 4, out_pages, None)
    return rc, lib.qmm_last_error().decode()


def test_read_refusals(capi):
    for what, text in ((dict(batch=-1), "non-negative"), (dict(pages=-1), "non-negative"), (dict(out_pages=-1), "non-negative"),
                       (dict(cache=_cache(capi, page_size=0)), "positive"), (dict(out=_cache(capi, page_size=0)), "positive"),
                       (dict(batch=2**31), "out of range"), (dict(out_pages=2**31), "out of range"), (dict(cache=_cache(capi, dim=257)), "up to 256"),
                       (dict(cache=_cache(capi, kv_heads=0)), "heads"), (dict(out=_cache(capi, dim=32)), "same heads and dimension"),
                       (dict(out=_cache(capi, kv_heads=3)), "same heads and dimension"), (dict(out_dtype=3), "bf16, f16 or f32"),
                       (dict(out=_cache(capi, value=1 << 20)), "same address"), (dict(scales=_scales(capi, key=1)), "4-byte"),
                       (dict(table=2), "4-byte"), (dict(out_table=2), "4-byte"), (dict(lens=3), "4-byte"), (dict(first=2), "4-byte"),
                       (dict(out=_cache(capi, key=1)), "its type"), (dict(out=_cache(capi, key=2), out_dtype=2), "its type")):
        rc, message = _read(capi, **what)
        assert rc == 1 and text in message, (what, message)
    assert _read(capi, batch=0)[0] == 0


def test_workspace_sizes(capi):
    """The scratch is bounded by the GPU, not by the batch or the cache."""
    lib, n = capi.lib(), ctypes.c_size_t(0)

    def size(*a):
        assert lib.qmm_paged_quant_attention_workspace_size(*a, ctypes.byref(n)) == 0
        return n.value

    assert size(0, 8, 2, 64, 100) == 0 and size(4, 0, 2, 64, 100) == 0
    assert size(1, 64, 8, 128, 1 << 20) == size(4096, 64, 8, 128, 1 << 20) <= 60 << 20
    assert lib.qmm_paged_quant_attention_workspace_size(-1, 8, 2, 64, 100, ctypes.byref(n)) == 1
    assert lib.qmm_paged_quant_attention_workspace_size(1, 8, 0, 64, 100, ctypes.byref(n)) == 1


def test_oracle_against_loops():
    """The oracle's rows and sums against the definition, element by element."""
    g = torch.Generator().manual_seed(3)
    y = torch.randn((3, 2, 16), generator=g, dtype=torch.float64)
    y[0, 0], y[1, 1, 3], y[2, 0, 2] = 0.0, math.nan, math.inf
    codes, scale = oracle.quantize(y)
    for t in range(3):
        for h in range(2):
            row = y[t, h].tolist()
            if any(math.isnan(x) for x in row):
                assert math.isnan(scale[t, h]) and not codes[t, h].any()
                continue
            want = torch.tensor(max(abs(x) for x in row) / 127, dtype=torch.float64).float()
            assert scale[t, h] == want
            s = float(want)
            assert codes[t, h].tolist() == ([round(x / s) for x in row] if 0 < s < math.inf else [0] * 16)
    k, v = (torch.randint(-128, 128, (5, 3, 2, 16), generator=g, dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.rand((5, 2, 3), generator=g) for _ in range(2))
    q = torch.randn((2, 4, 16), generator=g).bfloat16()
    table, lens = torch.tensor([[2, 0, 9], [4, -1, 1]], dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    out, lse, *_ = oracle.attention(q, k, v, ks, vs, table, lens, scale=0.01, window=3, sinks=1)
    for b, n in enumerate(lens.tolist()):
        for h in range(4):
            sums, total = [0.0] * 16, 0.0
            for j in range(n):
                at, i = int(table[b, j // 3]), j % 3
                if not (n - 1 - j < 3 or j < 1) or not 0 <= at < 5:
                    continue
                e = math.exp(0.01 * float(q[b, h].double() @ k[at, i, h // 2].double()) * float(ks[at, h // 2, i]))
                total += e
                sums = [s + e * float(x) * float(vs[at, h // 2, i]) for s, x in zip(sums, v[at, i, h // 2])]
            assert abs(float(lse[b, h]) - math.log(total)) < 1e-12
            assert all(abs(float(x) - s / total) < 1e-11 for x, s in zip(out[b, h], sums))
    k_out, v_out = oracle.read_back(k, v, ks, vs, table, lens, torch.zeros((3, 4, 2, 16)), torch.ones((3, 4, 2, 16)), torch.tensor([[1, 0], [2, 7]]),
                                    first=torch.tensor([1, 0]))
    assert torch.equal(k_out[1, 2], k[2, 2].float() * ks[2, :, 2, None]) and torch.equal(v_out[0, 0], v[0, 1].float() * vs[0, :, 1, None])
    assert not k_out[1, 0].any() and bool((v_out[2, 3] == 1).all()) and torch.equal(k_out[2, 2], k[4, 2].float() * ks[4, :, 2, None])


def test_batches_near_32_bits(capi):
    """A warp's count of sequences goes up to 32 beyond the last one."""
    for batch in (2**31 - 256 + 1, 2**31 - 2):
        for call in (_attention, _read):
            rc, message = call(capi, batch=batch)
            assert rc == 1 and "out of range" in message
