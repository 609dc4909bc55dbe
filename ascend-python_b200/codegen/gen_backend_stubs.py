"""yaml op registry -> C++ dispatch stubs and torch-library registration.

Plays the role of the reference's ``python -m codegen.gen_backend_stubs``
(codegen/gen_backend_stubs.py:7-74, codegen/gen.py:226-292): every ``func:``
entry of ``op_plugin_functions.yaml`` becomes

* a declaration ``OP_PLUGIN_HIDDEN <ret> <name>(<args with defaults>);`` in
  ``OpApiInterface.h`` (namespace ``op_api``) and ``OpInterface.h``
  (namespace ``op_plugin``),
* a dispatch body in ``OpInterface.cpp`` that forwards to the namespace named
  by ``impl_ns`` (only ``op_api`` exists here: there is one backend),

and — the step the reference leaves to its host framework — a
``TORCH_LIBRARY_FRAGMENT(npu, ...)`` definition plus a CUDA-key implementation
in ``TorchLibrary.cpp`` so that ``torch.ops.npu.<name>`` resolves.

The schema grammar handled is the subset these operators use:
``Tensor``, ``Tensor(a!)`` (written in place), ``Tensor?``, ``str``, ``int``, ``int[]``,
``float``, ``float?``, ``bool``, ``ScalarType?``, keyword-only marker ``*``, defaults, and
``Tensor`` / tuple-of-``Tensor`` returns.

Usage: ``python -m codegen.gen_backend_stubs --source_yaml <yaml> [<yaml> ...] --output_dir <dir>``
"""
from __future__ import annotations

import argparse
import re
from dataclasses import dataclass
from pathlib import Path
from typing import List, Optional

import yaml

CPP_ARG_TYPES = {
    "Tensor": "const at::Tensor &",
    "Tensor?": "const c10::optional<at::Tensor> &",
    "str": "c10::string_view",
    "int": "int64_t",
    "int[]": "at::IntArrayRef",
    "float": "double",
    "float?": "c10::optional<double>",
    "bool": "bool",
    "ScalarType?": "c10::optional<at::ScalarType>",
    "ScalarType": "at::ScalarType",
}


@dataclass
class Argument:
    type: str
    name: str
    default: Optional[str]
    kwarg_only: bool

    def cpp_default(self) -> Optional[str]:
        if self.default is None:
            return None
        d = self.default
        if d == "None":
            return "c10::nullopt"
        if d in ("True", "False"):
            return d.lower()
        if d == "[]":
            return "{}"
        if self.type == "str":
            return '"' + d.strip("'\"") + '"'
        return d

    def decl(self, with_default: bool) -> str:
        t = CPP_ARG_TYPES[self.type]
        sep = "" if t.endswith("&") else " "
        s = f"{t}{sep}{self.name}"
        d = self.cpp_default()
        if with_default and d is not None:
            s += f"={d}"
        return s


@dataclass
class OpSchema:
    name: str
    args: List[Argument]
    returns: List[str]
    impl_ns: List[str]
    schema: str

    def cpp_return(self) -> str:
        if len(self.returns) == 1:
            return "at::Tensor"
        return "::std::tuple<" + ",".join("at::Tensor" for _ in self.returns) + ">"

    def signature(self, with_defaults: bool, qualifier: str = "") -> str:
        args = ", ".join(a.decl(with_defaults) for a in self.args)
        return f"{self.cpp_return()} {qualifier}{self.name}({args})"

    def call_args(self) -> str:
        return ", ".join(a.name for a in self.args)


_FUNC_RE = re.compile(r"^\s*(?P<name>[A-Za-z_][A-Za-z0-9_\.]*)\((?P<args>.*)\)\s*->\s*(?P<ret>.+?)\s*$")


def parse_schema(func: str, impl_ns) -> OpSchema:
    m = _FUNC_RE.match(func)
    if not m:
        raise ValueError(f"cannot parse schema: {func}")
    args: List[Argument] = []
    kwarg_only = False
    for raw in [a.strip() for a in m.group("args").split(",") if a.strip()]:
        if raw == "*":
            kwarg_only = True
            continue
        default = None
        if "=" in raw:
            raw, default = [p.strip() for p in raw.split("=", 1)]
        parts = raw.split()
        if len(parts) != 2:
            raise ValueError(f"cannot parse argument '{raw}' in: {func}")
        typ, name = parts
        typ = re.sub(r"^Tensor\([a-z]!\)$", "Tensor", typ)
        if typ not in CPP_ARG_TYPES:
            raise ValueError(f"unsupported argument type '{typ}' in: {func}")
        args.append(Argument(typ, name, default, kwarg_only))
    ret = m.group("ret").strip()
    if ret.startswith("("):
        returns = [r.strip() for r in ret.strip("()").split(",") if r.strip()]
    else:
        returns = [ret]
    if any(r != "Tensor" for r in returns):
        raise ValueError(f"unsupported return type in: {func}")
    if isinstance(impl_ns, str):
        impl_ns = [s.strip() for s in impl_ns.split(",")]
    return OpSchema(m.group("name"), args, returns, list(impl_ns or []), func.strip())


def parse_native_yaml(path) -> List[OpSchema]:
    """Sections follow the reference registry: ``official``, ``symint``, ``custom``
    (codegen/gen.py:196-212); all three keys must be present."""
    with open(path, "r") as f:
        es = yaml.safe_load(f)
    for key in ("symint", "official", "custom"):
        if key not in es:
            raise AssertionError(f"Can't find {key} in yaml.")
    ops = []
    for e in (es["official"] or []) + (es["custom"] or []):
        ops.append(parse_schema(e["func"], e.get("impl_ns")))
    return ops


HEADER = """// Generated by codegen/gen_backend_stubs.py from op_plugin/config/op_plugin_functions.yaml.
// Do not edit.
"""


def gen_interface_header(ops: List[OpSchema], namespace: str, guard: str) -> str:
    decls = "\n".join(f"OP_PLUGIN_HIDDEN {op.signature(True)};" for op in ops)
    return f"""{HEADER}#ifndef {guard}
#define {guard}

#include <ATen/ATen.h>
#include <c10/util/Optional.h>
#include <c10/util/string_view.h>
#include <tuple>

#include "op_plugin/utils/Export.h"

namespace {namespace} {{
{decls}
}}  // namespace {namespace}
#endif  // {guard}
"""


def gen_dispatch(ops: List[OpSchema]) -> str:
    bodies = []
    for op in ops:
        if op.impl_ns != ["op_api"]:
            raise AssertionError(f"unknown namespace {op.impl_ns} for {op.name}: this build has the op_api backend only")
        bodies.append(f"""{op.signature(False)}
{{
    return op_api::{op.name}({op.call_args()});
}}
""")
    body = "\n".join(bodies)
    return f"""{HEADER}#include "op_plugin/OpApiInterface.h"
#include "op_plugin/OpInterface.h"

namespace op_plugin {{
{body}}}  // namespace op_plugin
"""


def gen_torch_library(ops: List[OpSchema]) -> str:
    defs = "\n".join(f'    m.def("{op.schema}");' for op in ops)
    impls = "\n".join(f'    m.impl("{op.name}", TORCH_FN(op_plugin::{op.name}));' for op in ops)
    return f"""{HEADER}#include <torch/library.h>

#include "op_plugin/OpInterface.h"

// Schemas live in the `npu` namespace so that call sites written against the
// reference (`torch.ops.npu.<op>` / `torch_npu.<op>`) resolve unchanged.
TORCH_LIBRARY_FRAGMENT(npu, m)
{{
{defs}
}}

TORCH_LIBRARY_IMPL(npu, CUDA, m)
{{
{impls}
}}
"""


def _write_if_changed(path: Path, text: str) -> None:
    if path.exists() and path.read_text() == text:
        return
    path.write_text(text)


def run(source_yaml, output_dir) -> List[OpSchema]:
    """``source_yaml``: one registry or a list of them."""
    sources = source_yaml if isinstance(source_yaml, (list, tuple)) else [source_yaml]
    ops = [op for source in sources for op in parse_native_yaml(source)]
    out = Path(output_dir)
    _write_if_changed(out / "OpApiInterface.h", gen_interface_header(ops, "op_api", "OP_PLUGIN_OPAPI_INTERFACE_H_"))
    _write_if_changed(out / "OpInterface.h", gen_interface_header(ops, "op_plugin", "OP_PLUGIN_OP_INTERFACE_H_"))
    _write_if_changed(out / "OpInterface.cpp", gen_dispatch(ops))
    _write_if_changed(out / "TorchLibrary.cpp", gen_torch_library(ops))
    return ops


def main() -> None:
    parser = argparse.ArgumentParser(description="Generate op_plugin dispatch stubs")
    parser.add_argument("-s", "--source_yaml", required=True, nargs="+")
    parser.add_argument("-o", "--output_dir", required=True)
    opts = parser.parse_args()
    run(opts.source_yaml, opts.output_dir)


if __name__ == "__main__":
    main()
