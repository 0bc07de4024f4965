"""Writes ``rust/cleave_cuda_sys.rs``: the Rust side of the C ABI that a cleave maintainer adds to the
compiler -- one ``extern "C"`` declaration per function of ``include/cleave_cuda.h`` and one
``register_symbol`` line per function for the JIT (cleave/src/pipeline.rs:159-198 registers the
runtime's symbols the same way).  Types come from the ctypes table of ``cleave_b200/_lib.py``
(which a test keeps equal to the header), parameter names from the header.

    python cleave_b200/cleave/gen_rust_bindings.py            # rewrite the file
    python cleave_b200/cleave/gen_rust_bindings.py --check    # exit 1 if the file is stale
"""
from __future__ import annotations

import ctypes
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
OUT = os.path.join(HERE, "rust", "cleave_cuda_sys.rs")


def rust_type(t) -> str:
    if t is None:
        return "()"
    table = {ctypes.c_int32: "i32", ctypes.c_int64: "i64", ctypes.c_float: "f32", ctypes.c_double: "f64",
             ctypes.c_uint32: "u32", ctypes.c_uint64: "u64", ctypes.c_uint8: "u8",
             ctypes.c_void_p: "*mut c_void", ctypes.c_char_p: "*const c_char"}
    if t in table:
        return table[t]
    if isinstance(t, type) and issubclass(t, ctypes._Pointer):
        return "*mut " + rust_type(t._type_)
    raise TypeError(f"no Rust spelling for {t!r}")


def header_param_names() -> dict[str, list[str]]:
    with open(os.path.join(ROOT, "include", "cleave_cuda.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    names = {}
    for fn, params in re.findall(r"\b(cleave_cuda_\w+)\s*\(([^)]*)\)\s*;", text):
        ps = [p.strip() for p in params.split(",") if p.strip() and p.strip() != "void"]
        names[fn] = [re.sub(r"\[.*\]$", "", p.split()[-1].lstrip("*")) for p in ps]
    return names


def render() -> str:
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    from cleave_b200._lib import SIGNATURES
    names = header_param_names()
    out = ["// Generated by cleave_b200/cleave/gen_rust_bindings.py from include/cleave_cuda.h -- do not edit.",
           "// Rust declarations of libcleave_cuda and the JIT registration of its symbols.",
           "// Not compiled where it was generated (no Rust toolchain there).",
           "#![allow(non_snake_case)]",
           "use std::os::raw::{c_char, c_void};",
           "",
           '#[link(name = "cleave_cuda")]',
           'unsafe extern "C" {']
    for fn, (res, args) in SIGNATURES.items():
        pn = names.get(fn, [])
        ps = ", ".join(f"{pn[i] if i < len(pn) else f'a{i}'}: {rust_type(t)}" for i, t in enumerate(args))
        ret = "" if res is None else f" -> {rust_type(res)}"
        out.append(f"    pub fn {fn}({ps}){ret};")
    out += ["}", "",
            "/// Call beside `register_cleave_rt_symbols` so that `func.call @cleave_cuda_*` resolves in the JIT.",
            "pub fn register_cleave_cuda_symbols(engine: &melior::ExecutionEngine) {",
            "    unsafe {"]
    for fn in SIGNATURES:
        out.append(f'        engine.register_symbol("{fn}", {fn} as *mut ());')
    out += ["    }", "}", ""]
    return "\n".join(out)


def main() -> int:
    text = render()
    if "--check" in sys.argv:
        try:
            with open(OUT) as f:
                return 0 if f.read() == text else 1
        except OSError:
            return 1
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    with open(OUT, "w") as f:
        f.write(text)
    print("wrote", OUT)
    return 0


if __name__ == "__main__":
    sys.exit(main())
